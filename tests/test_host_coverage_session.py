"""The launch shape coverage test is skipped in a session that lacks a module whose cases reach shapes of their own."""
from __future__ import annotations

import types

import conftest


class Item:
    def __init__(self, module):
        self.module, self.markers = types.SimpleNamespace(__name__=module), []

    def add_marker(self, marker):
        self.markers.append(marker)


def test_a_session_without_a_module_skips_the_coverage_test_alone():
    for present in ((), ("test_gpu_attention",), conftest.COVERAGE_MODULES):
        items = [Item(name) for name in ("test_gpu_rope", *present, "test_zy_launch_shape_coverage")]
        conftest.pytest_collection_modifyitems(items)
        assert not any(item.markers for item in items[:-1])
        assert [marker.name for marker in items[-1].markers] == ([] if present == conftest.COVERAGE_MODULES else ["skip"])
