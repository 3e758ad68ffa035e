"""Attention of so many rows, heads or sequences that one axis of a grid, which counts threads in 32 bits, does not hold its
blocks.  The sequences are a key or two long, so that what has to come out is known in closed form."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyle_amd import compute as hc
from hyle_amd import torch_io as tio

from attention_support import assert_within, attention_rows
from gpu_support import DEVICE, context, note

pytestmark = pytest.mark.gpu


def random(seed, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(0.0, std, generator=torch.Generator(DEVICE).manual_seed(seed))


def launch(operation, inputs):
    bound = tio.Bound(context(), operation, [tio.desc_of(t) for t in inputs])
    outputs = [t.fill_(77.0) for t in bound.outputs()]
    bound.submit(inputs, outputs)
    torch.cuda.synchronize()
    return outputs


def assert_one_key(scale, query, key, value, outputs):
    """Rows that see one key [..., heads, 1, depth] (queries [..., heads, shared, depth]): its weight is exp(0) / exp(0), so the
    output is its value; the logarithm is the score, off by depth + 2 roundings of the sum of its terms' sizes, those of the power
    of two and its logarithm (2^-20) and two of its own."""
    out, logs = outputs[0].view(query.shape), outputs[1].view(query.shape[:-1])
    assert torch.equal(out, value.expand(query.shape))
    terms = query.double() * key.double() * scale
    bound = (query.shape[-1] + 4) * 2.0 ** -24 * terms.abs().sum(-1) + 2.0 ** -20
    assert ((logs.double() - terms.sum(-1)).abs() <= bound).all()


@pytest.mark.parametrize("rows", [63, 64, 65])
def test_f32_rows_and_heads_past_a_grids_axis(rows):
    """Blocks of 512 threads, one to a row and head: 2^23 of them are 2^32 threads.  Two keys: sigmoids in closed form."""
    batch, queries, depth = 2 ** 13, 16, 4
    q, k, v = random(1, (batch, rows, queries, depth), torch.float32), random(2, (batch, 2, 1, depth), torch.float32), random(3, (batch, 2, 1, depth), torch.float32)
    note(f"f32 attention of {batch} x {rows} rows of {queries} heads")
    (out,) = launch(hc.Attention(0.5, False), [q, k, v])
    assert hc.last_launch_variant() == "attention_rows"
    for part in range(0, batch, 1024):
        span = slice(part, part + 1024)
        terms = 0.5 * q[span, :, :, None].double() * k[span, None, None, :, 0].double()  # [batch, rows, heads, keys, depth]
        score = terms.sum(-1)
        weight = torch.softmax(score, -1)[..., None] * v[span, None, None, :, 0].double()
        # a score is off by depth + 2 roundings of its terms' sizes and 4 of its own (the power), so the weights by twice e, and
        # the two products, their sum and the division by 8 roundings
        e = 10 * 2.0 ** -24 * terms.abs().sum(-1).amax(-1) + 2.0 ** -20
        bound = (4 * e[..., None] + 8 * 2.0 ** -24) * weight.abs().sum(-2)
        assert ((out[span].double() - weight.sum(-2)).abs() <= bound).all()


def test_packed_sequences_past_a_grids_axis():
    """Blocks of 256 threads, one to a sequence and head: 2^24 of them are 2^32 threads."""
    sequences, queries, depth = 2 ** 20 + 2 ** 14, 16, 8
    q, k, v = random(4, (sequences, queries, depth), torch.float16), random(5, (sequences, 1, depth), torch.float16), random(6, (sequences, 1, depth), torch.float16)
    marks = torch.arange(sequences + 1, dtype=torch.int32, device=DEVICE)
    note(f"packed attention of {sequences} sequences of {queries} heads")
    outputs = launch(hc.Attention(0.3, return_log_sum=True), [q, k, v, marks])
    assert hc.last_launch_variant() == "attention_rows"
    assert_one_key(0.3, q, k, v, outputs)


@pytest.mark.parametrize("batch", [2 ** 22 - 1, 2 ** 22])
def test_a_batch_of_single_keys_past_a_grids_axis(batch):
    q, k, v = (random(7 + i, (batch, 1, 4, 8), torch.bfloat16) for i in range(3))
    note(f"attention of {batch} sequences of one key")
    outputs = launch(hc.Attention(0.3, return_log_sum=True), [q, k, v])
    assert hc.last_launch_variant() == ("attention_split/below-d64/16-rows" if batch % 2 else "attention_rows")
    assert_one_key(0.3, q, k, v, outputs)


@pytest.mark.parametrize("batch", [2 ** 22 - 1, 2 ** 22])
def test_a_paged_batch_past_a_grids_axis(batch):
    """One key or none to a sequence, on pages that many of them share."""
    pages, heads, depth = 100, 4, 8
    query, cache = random(10, (batch, heads, depth), torch.bfloat16), random(11, (pages, 2, heads, 1, depth), torch.bfloat16)
    table = torch.randint(0, pages, (batch, 1), device=DEVICE, generator=torch.Generator(DEVICE).manual_seed(12)).to(torch.int32)
    lengths = (torch.arange(batch, device=DEVICE) % 5 != 3).to(torch.int32)
    note(f"paged attention of {batch} sequences")
    out, logs = launch(hc.PagedAttention(0.3, return_log_sum=True), [query, cache, table, lengths])
    assert hc.last_launch_variant() == ("attention_split/below-d64/16-rows" if batch % 2 else "attention_rows")
    empty = lengths == 0
    assert (out[empty] == 0).all() and (logs[empty] == -np.inf).all()
    some = ~empty
    held = cache[table[some, 0].long()]
    assert_one_key(0.3, query[some][:, :, None], held[:, 0], held[:, 1], [out[some], logs[some]])


@pytest.mark.parametrize("sequences", [64, 65, 4096, 4097, 70001, 2 ** 20 - 1])
def test_packed_sequences_are_found_among_any_number_of_them(sequences):
    """Sequences of no, one and, in places, some hundred rows: every tile finds its own."""
    rng, queries = np.random.default_rng(sequences), 2 if sequences < 2 ** 17 else 16
    lengths = rng.integers(0, 2, sequences)
    for i, rows in ((0, 130), (sequences // 2, 300), (sequences - 1, 129)):
        lengths[i] = rows
    offsets = np.concatenate([[3], 3 + np.cumsum(lengths)]).astype(np.int32)
    rows = int(offsets[-1]) + 5
    q, k, v = (random(20 + i, (rows, heads, 8), torch.bfloat16) for i, heads in enumerate((queries, 1, 1)))
    operation = hc.Attention(0.3, return_log_sum=True)
    note(f"packed attention of {sequences} sequences")
    outputs = launch(operation, [q, k, v, torch.from_numpy(offsets).to(DEVICE)])
    assert hc.last_launch_variant().startswith("attention_tiles/d64/")
    single = np.repeat(lengths, lengths) == 1
    alone = torch.from_numpy(3 + np.flatnonzero(single)).to(DEVICE)
    assert_one_key(0.3, q[alone][:, None], k[alone][:, None], v[alone][:, None], [t[alone] for t in outputs])
    for i in (0, sequences // 2, sequences - 1):
        span = slice(int(offsets[i]), int(offsets[i + 1]))
        out, logs, bound, log_bound = attention_rows(*(t[span].double().cpu().numpy() for t in (q, k, v)), 0, True, 0, 0, 0.3, torch.bfloat16)
        assert_within(outputs[0][span], out, bound)
        assert_within(outputs[1][span], logs, log_bound)
    for t in outputs:
        assert (t[:3] == 77.0).all() and (t[-5:] == 77.0).all()


def test_eight_times_the_sequences_take_about_eight_times_as_long():
    """Not sixty-four times, as they do where every block looks through all sequences."""
    def best(sequences):
        q, k, v = (random(30 + i, (sequences, heads, 64), torch.bfloat16) for i, heads in enumerate((8, 2, 2)))
        marks = torch.arange(sequences + 1, dtype=torch.int32, device=DEVICE)
        bound = tio.Bound(context(), hc.Attention(0.125), [tio.desc_of(t) for t in (q, k, v, marks)])
        outputs, times = bound.outputs(), []
        for _ in range(6):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            bound.submit([q, k, v, marks], outputs)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)
    note("packed attention of 4096 and of 32768 sequences")
    assert best(2 ** 15) < 24 * best(2 ** 12)
