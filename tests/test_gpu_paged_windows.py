"""PagedAttention whose windows and sinks are dealt to several chunks and joined, and chunks of prompts over a paged cache: new
tokens by the hundred, some of which see nothing of what others see."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyle_amd import compute as hc

from gpu_support import note
from test_gpu_paged_attention import TYPES, Paged, attend, check, values

pytestmark = pytest.mark.gpu

LENGTHS = [9000, 500, 0, 3001, 2050, 1]


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [2048, 777])
@pytest.mark.parametrize("sinks", [0, 4, 130, 1500])
@pytest.mark.parametrize("new,shared", [(1, 4), (4, 4), (4, 8), (4, 16)])
def test_windows_of_several_chunks(cache, window, sinks, new, shared):
    """16, 32 and 64 rows to a block; windows that begin between two tiles behind sinks that end inside one."""
    rng = np.random.default_rng(window + sinks + new * shared)
    paged = Paged(rng, LENGTHS, 1, 64, 16, TYPES[cache])
    query = values(rng, (len(LENGTHS), new, shared, 64), torch.bfloat16, 1.5)
    operation = hc.PagedAttention(0.125, window, sinks, True)
    note(f"paged attention {cache}, window {window}, sinks {sinks}, {new} x {shared} rows, joined")
    check(operation, query, paged, LENGTHS, attend(operation, query, paged))
    rows = 16 if new * shared <= 16 else 32 if new * shared <= 32 else 64
    assert f"/{rows}-rows + attention_join" in hc.last_launch_variant()


@pytest.mark.parametrize("depth", [80, 128, 256])
@pytest.mark.parametrize("window,sinks", [(2048, 4), (777, 130)])
def test_windows_of_several_chunks_at_other_depths(depth, window, sinks):
    rng = np.random.default_rng(depth + window)
    paged = Paged(rng, LENGTHS, 2, depth, 24, torch.float16)
    query = values(rng, (len(LENGTHS), 2, 8, depth), torch.float16, 1.5)
    operation = hc.PagedAttention(depth ** -0.5, window, sinks, True)
    note(f"paged attention of depth {depth}, window {window}, sinks {sinks}, joined")
    check(operation, query, paged, LENGTHS, attend(operation, query, paged))
    assert "attention_join" in hc.last_launch_variant()


@pytest.mark.parametrize("window,sinks", [(600, 0), (640, 33), (2048, 4), (3000, 700)])
@pytest.mark.parametrize("length", [608, 640, 672, 3001, 6000])
def test_one_sequence_under_a_window(window, sinks, length):
    """Lengths at which the sinks' tiles and the window's are one more than the tiles of all keys."""
    rng = np.random.default_rng(window + length)
    paged = Paged(rng, [length], 1, 64, 16, torch.bfloat16)
    query = values(rng, (1, 2, 4, 64), torch.bfloat16, 1.5)
    operation = hc.PagedAttention(0.125, window, sinks, True)
    note(f"paged attention of one sequence of {length}, window {window}, sinks {sinks}")
    check(operation, query, paged, [length], attend(operation, query, paged))
    assert "attention_join" in hc.last_launch_variant()


@pytest.mark.parametrize("window,sinks", [(700, 5), (1500, 200)])
def test_many_sequences_under_a_window(window, sinks):
    """More than the 64 that a wave looks at together, of every length; and so many that a chunk is several tiles."""
    rng = np.random.default_rng(window)
    lengths = [int(n) for n in rng.integers(0, 3000, 150)]
    paged = Paged(rng, lengths, 8, 64, 16, torch.bfloat16)
    query = values(rng, (len(lengths), 8, 64), torch.bfloat16, 1.5)
    operation = hc.PagedAttention(0.125, window, sinks, True)
    note(f"paged attention of 150 sequences, window {window}, sinks {sinks}")
    check(operation, query, paged, lengths, attend(operation, query, paged))
    assert "attention_join" in hc.last_launch_variant()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("depth", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (128, 0), (150, 3)])
@pytest.mark.parametrize("new,queries", [(300, 2), (513, 1)])
def test_chunks_of_prompts_over_a_cache(cache, depth, window, sinks, new, queries):
    """Behind a prefix, alone, and more new tokens than the sequence has."""
    rng, lengths = np.random.default_rng(depth + new), [1500, new, 200, 0]
    paged = Paged(rng, lengths, 1, depth, 16, TYPES[cache])
    query = values(rng, (len(lengths), new, queries, depth), torch.bfloat16, 1.5)
    operation = hc.PagedAttention(depth ** -0.5, window, sinks, True)
    note(f"paged attention of {new} new tokens {cache} depth {depth}, window {window}, sinks {sinks}")
    check(operation, query, paged, lengths, attend(operation, query, paged))
