"""Attention whose scale makes up for queries and keys of other sizes: it multiplies their products, which f32 holds, not the
queries, which it would not."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyle_amd import compute as hc
from hyle_amd import torch_io as tio

from attention_support import assert_within, attention_rows
from gpu_support import DEVICE, context, note

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("tag", ["f32", "bf16"])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("q_size,k_size,scale", [(1e30, 1e-30, 0.3), (1e30, 2e-38, 1e9), (1e-30, 1e37, 3e-8), (4.0, 2e-38, 2.0 ** 126), (1e-12, 1e37, 1e-25)])
def test_scales_of_any_size(tag, aligned, q_size, k_size, scale):
    rng, dtype = np.random.default_rng(5), TYPES[tag]
    def values(rows, heads, size):
        x = rng.normal(0, 1, 1 + rows * heads * 16)
        x = torch.from_numpy((x + np.sign(x)) * size).to(DEVICE).to(torch.float32).to(dtype)  # (no subnormals)
        return (x[:-1] if aligned else x[1:]).view(rows, heads, 16)
    q, k, v = values(90, 2, q_size), values(90, 1, k_size), values(90, 1, 1.0)
    q[3], k[0] = 0.0, 0.0
    operation = hc.Attention(scale, return_log_sum=True)
    bound = tio.Bound(context(), operation, [tio.desc_of(t) for t in (q, k, v)])
    outputs = bound.outputs()
    note(f"attention of queries of {q_size}, keys of {k_size}, scale {scale} {tag} {aligned}")
    bound.submit([q, k, v], outputs)
    torch.cuda.synchronize()
    held = float(np.float32(scale))
    out, logs, out_bound, log_bound = attention_rows(*(t.double().cpu().numpy() for t in (q, k, v)), 0, True, 0, 0, held, dtype)
    assert_within(outputs[0], out, out_bound)
    assert_within(outputs[1], logs, log_bound)
