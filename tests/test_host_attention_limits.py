"""What attention plans ask for at the limits of a launch, without a device."""
from __future__ import annotations

import pytest

from hyle_amd import compute as hc

DT, D = hc.DataType, hc.TensorDesc.dense
CTX = hc.Context.planning_only()
BF16, I32 = DT.kBFloat16, DT.kInt32


def test_a_split_whose_blocks_no_grid_holds_is_not_planned():
    """256 threads to a block: 2^24 blocks are one too many."""
    def plan(sequences):
        return hc.prepare(CTX, hc.PagedAttention(), D(BF16, [sequences, 4, 8]), D(BF16, [64, 2, 4, 16, 8]), D(I32, [sequences, 64]), D(I32, [sequences]))
    fits, past = plan(2 ** 22 - 2 ** 14), plan(2 ** 22)
    assert fits.dispatch_count() == 2 and fits.workspace_requirement().size > 0
    assert past.dispatch_count() == 1 and past.workspace_requirement().size == 0


def test_more_pages_than_slots_can_count_are_refused():
    """Also where the low 64 bits of the number are few."""
    keys = D(BF16, [3, 4, 64])
    for pages in (2 ** 31, 2 ** 64 + 10):
        with pytest.raises(hc.StatusError) as refused:
            hc.infer_output_descriptions(hc.PagedAppend(pages, 1, BF16), [keys, keys, D(I32, [3])])
        assert refused.value.is_invalid_argument()


def test_scales_whose_base_two_logarithms_pass_f32_are_declined():
    q, cache = D(BF16, [2, 4, 64]), D(BF16, [8, 2, 4, 16, 64])
    for scale in (2.0 ** 127, -2.0 ** 127):
        assert hc.prepare(CTX, hc.Attention(scale), q, q, q).dispatch_count() == 1
    for scale in (2.4e38, -3e38):
        for operation, inputs in ((hc.Attention(scale), (q, q, q)), (hc.PagedAttention(scale), (q, cache, D(I32, [2, 3]), D(I32, [2])))):
            with pytest.raises(hc.StatusError) as refused:
                hc.prepare(CTX, operation, *inputs)
            assert refused.value.code == hc.StatusCode.kUnimplemented
