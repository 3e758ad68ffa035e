"""Batches of few rows to a key head: as many of them as leave compute units idle, and more than fill the device."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyle_amd import compute as hc

from gpu_support import note
from test_gpu_attention import TYPES, check_batched, launch, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tag,depth", [("bf16", 64), ("f16", 80), ("bf16", 128), ("f16", 256)])
@pytest.mark.parametrize("batch,shared", [(12, 4), (70, 4), (70, 2), (70, 1)])
@pytest.mark.parametrize("rows,keys", [(8, 60), (16, 300)])
def test_few_rows_of_many_sequences(tag, depth, batch, shared, rows, keys):
    rng = np.random.default_rng(depth + batch + rows)
    q, k, v = (values(rng, (batch, n, heads, depth), TYPES[tag], std) for n, heads, std in ((rows, 4 * shared, 1.5), (keys, 4, 1.0), (keys, 4, 1.0)))
    lengths = [int(n) for n in rng.integers(0, keys + 1, batch)]
    marks = torch.tensor(lengths, dtype=torch.int32, device=q.device)
    note(f"attention of {batch} sequences of {rows} x {shared} rows over {keys} keys {tag} {depth}")
    for operation in (hc.Attention(depth ** -0.5, return_log_sum=True), hc.Attention(depth ** -0.5, False)):
        check_batched(operation, TYPES[tag], q, k, v, lengths, launch(operation, [q, k, v, marks]))


@pytest.mark.parametrize("shared", [2, 4])
def test_tiles_that_would_take_turns_over_the_same_keys_are_split(shared):
    """64 rows to a key head behind 512 keys of 40 x 8 key heads: the tiles took up to 2.7 times as long."""
    rng = np.random.default_rng(shared)
    q, k, v = (values(rng, (40, n, heads, 128), torch.bfloat16) for n, heads in ((64 // shared, 8 * shared), (512, 8), (512, 8)))
    operation = hc.Attention(0.088, False)
    note(f"attention of 40 sequences of 64 rows to a key head, {shared} query heads to it")
    outputs = launch(operation, [q, k, v])
    assert hc.last_launch_variant().startswith("attention_split/")
    check_batched(operation, torch.bfloat16, q[:3], k[:3], v[:3], None, [outputs[0][:3]])
