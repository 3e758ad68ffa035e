"""Attention against the definition in 64 bits: packed and padded batches, windows with sinks, rows that see nothing, odd
depths, lengths and strides, values that are no numbers where a row does not look, and the calls that a launch refuses."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from hyle_amd import compute as hc
from hyle_amd import torch_io as tio

from attention_support import assert_within, attention_rows
from gpu_support import DEVICE, context, note

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNTOUCHED = 77.0


def values(rng, shape, dtype, std=1.0):
    return torch.from_numpy(rng.normal(0, std, shape).astype(np.float32)).to(DEVICE).to(dtype)


def host(tensor):
    return tensor.double().cpu().numpy()


def launch(operation, inputs):
    """One submit into outputs that hold another number before."""
    bound = tio.Bound(context(), operation, [tio.desc_of(t) for t in inputs])
    outputs = [t.fill_(UNTOUCHED) for t in bound.outputs()]
    bound.submit(inputs, outputs)
    torch.cuda.synchronize()
    return outputs


def check_packed(operation, dtype, q, k, v, offsets, outputs):
    """Every sequence's rows within their bounds, and the rows of none as they were."""
    marks = [min(max(m, 0), q.shape[0]) for m in offsets]
    owned = np.zeros(q.shape[0], bool)
    hq, hk, hv = host(q), host(k), host(v)
    for a, b in zip(marks[:-1], marks[1:]):
        owned[a:b] = True
        out, logs, bound, log_bound = attention_rows(hq[a:b], hk[a:b], hv[a:b], 0, operation.causal, operation.window, operation.sinks,
                                                     operation.scale, dtype)
        assert_within(outputs[0][a:b], out, bound)
        if operation.return_log_sum:
            assert_within(outputs[1][a:b], logs, log_bound)
    for t in outputs:
        assert (t[torch.from_numpy(~owned).to(DEVICE)] == UNTOUCHED).all(), "a row of no sequence was written"


def check_batched(operation, dtype, q, k, v, lengths, outputs):
    hq, hk, hv = host(q), host(k), host(v)
    for i in range(q.shape[0]):
        n = k.shape[1] if lengths is None else min(max(lengths[i], 0), k.shape[1])
        out, logs, bound, log_bound = attention_rows(hq[i], hk[i, :n], hv[i, :n], k.shape[1] - q.shape[1], operation.causal, operation.window,
                                                     operation.sinks, operation.scale, dtype)
        assert_within(outputs[0][i], out, bound)
        if operation.return_log_sum:
            assert_within(outputs[1][i], logs, log_bound)


# type, depth, query heads, key heads, offsets, rows, causal, window, sinks, scale, logarithms
PACKED = [
    ("bf16", 128, 4, 1, [0, 1], 1, True, 0, 0, 0.088, True),                         # one token
    ("bf16", 128, 2, 2, [0, 130], 130, True, 0, 0, 0.088, True),                     # just past a tile of 128 rows
    ("f16", 64, 4, 2, [0, 63, 64, 64, 200], 200, True, 0, 0, 0.125, False),          # one token and none among others
    ("bf16", 80, 5, 1, [3, 40, 171], 180, True, 0, 0, 0.11, True),                   # rows before the first and behind the last
    ("f16", 96, 3, 3, [0, 257], 257, False, 0, 0, 0.1, True),                        # not causal
    ("bf16", 256, 2, 1, [0, 100, 165], 165, True, 0, 0, 0.0625, True),               # the deepest
    ("f16", 128, 2, 1, [0, 300], 300, True, 33, 0, 0.088, True),                     # a window
    ("bf16", 128, 2, 1, [0, 400], 400, True, 65, 4, 0.088, True),                    # and first tokens that stay visible
    ("bf16", 64, 2, 2, [0, 290], 290, True, 1, 0, 0.125, False),                     # a query sees itself alone
    ("f16", 64, 2, 2, [0, 290], 290, True, 64, 100, 0.125, True),                    # sinks past a tile, overlapping the window
    ("bf16", 64, 1, 1, [0, 200], 200, True, 2 ** 31 - 1, 2 ** 31 - 1, 0.125, False),  # a window that hides nothing
    ("bf16", 32, 2, 1, [0, 150], 150, True, 0, 0, 0.0, True),                        # every weight alike
    ("bf16", 72, 2, 1, [0, 150], 150, True, 0, 0, -0.12, True),                      # a negative scale
    ("f16", 8, 2, 1, [0, 150], 150, True, 0, 0, 0.35, True),
    ("bf16", 63, 2, 1, [0, 140], 140, True, 0, 0, 0.12, True),                       # no whole vectors
    ("f16", 1, 3, 1, [0, 70], 70, True, 0, 0, 1.0, True),
    ("f32", 64, 2, 1, [0, 140], 140, True, 50, 2, 0.125, True),
    ("bf16", 128, 2, 1, [-5, 50, 50, 1000], 120, True, 0, 0, 0.088, False),          # marks outside: clamped
]


@pytest.mark.parametrize("case", PACKED, ids=[f"{c[0]}-d{c[1]}-{c[2]}x{c[3]}-{c[5]}rows-w{c[7]}s{c[8]}-{i}" for i, c in enumerate(PACKED)])
def test_packed_sequences(case):
    tag, depth, queries, heads, offsets, rows, causal, window, sinks, scale, logs = case
    dtype, rng = TYPES[tag], np.random.default_rng(depth * 1000 + rows)
    q, k, v = values(rng, (rows, queries, depth), dtype, 1.5), values(rng, (rows, heads, depth), dtype), values(rng, (rows, heads, depth), dtype)
    operation = hc.Attention(scale, causal, window, sinks, logs)
    note(f"packed attention {case}")
    marks = torch.tensor(offsets, dtype=torch.int32, device=DEVICE)
    check_packed(operation, dtype, q, k, v, offsets, launch(operation, [q, k, v, marks]))


# type, depth, query heads, key heads, batch, queries, keys, lengths, causal, window, sinks, logarithms
BATCHED = [
    ("bf16", 64, 4, 4, 3, 70, 70, [70, 0, 33], False, 0, 0, True),       # an encoder's batch, one of it empty
    ("f16", 128, 4, 2, 2, 40, 200, None, True, 0, 0, True),              # a chunk behind a prefix
    ("bf16", 128, 4, 1, 2, 1, 333, [333, 100], True, 0, 0, False),       # one query
    ("bf16", 128, 2, 1, 2, 50, 20, None, True, 0, 0, True),              # more queries than keys: the first see nothing
    ("f16", 80, 3, 1, 2, 130, 300, [300, 170], True, 64, 3, True),
    ("bf16", 256, 4, 2, 1, 3, 1000, None, True, 0, 0, True),
    ("bf16", 128, 8, 2, 1, 1, 3000, None, True, 0, 0, True),             # a long axis and one row
    ("f16", 64, 2, 2, 2, 20, 90, [-4, 1000], False, 0, 0, True),         # lengths outside: clamped
    ("bf16", 64, 2, 1, 2, 30, 0, None, True, 0, 0, True),                # no key at all
    ("f32", 40, 2, 1, 2, 9, 30, [30, 7], False, 0, 0, True),
]


@pytest.mark.parametrize("case", BATCHED, ids=[f"{c[0]}-d{c[1]}-{c[2]}x{c[3]}-{c[5]}of{c[6]}-{i}" for i, c in enumerate(BATCHED)])
def test_batched_sequences(case):
    tag, depth, queries, heads, batch, rows, keys, lengths, causal, window, sinks, logs = case
    dtype, rng = TYPES[tag], np.random.default_rng(depth * 100 + rows + keys)
    q, k, v = values(rng, (batch, rows, queries, depth), dtype, 1.5), values(rng, (batch, keys, heads, depth), dtype), values(rng, (batch, keys, heads, depth), dtype)
    operation = hc.Attention(depth ** -0.5, causal, window, sinks, logs)
    note(f"batched attention {case}")
    marks = [] if lengths is None else [torch.tensor(lengths, dtype=torch.int32, device=DEVICE)]
    check_batched(operation, dtype, q, k, v, lengths, launch(operation, [q, k, v, *marks]))


# as BATCHED, with enough tiles that a device is full of them: one wave to 32 rows instead of two
MANY = [
    ("bf16", 64, 8, 4, 40, 150, 150, None, True, 0, 0, True),
    ("f16", 80, 8, 2, 40, 150, 170, None, True, 40, 3, True),
    ("bf16", 128, 8, 2, 40, 150, 150, [150, 0, 129, 77] * 10, False, 0, 0, True),
    ("f16", 256, 8, 2, 20, 150, 150, None, True, 0, 0, True),
]


@pytest.mark.parametrize("case", MANY, ids=[f"{c[0]}-d{c[1]}-{c[4]}x{c[2]}" for c in MANY])
def test_many_sequences(case):
    test_batched_sequences(case)
    want = "/128x2x32" if case[1] == 256 else "/128x1x64"
    assert hc.last_launch_variant().endswith(want), hc.last_launch_variant()


def test_the_shape_of_a_tile_follows_the_blocks():
    rng = np.random.default_rng(8)
    for depth, rows, want in ((64, 60, "d64/128x1x64"), (64, 200, "d64/128x2x64"), (96, 60, "d96/128x1x64"), (96, 200, "d96/128x2x64"),
                              (128, 60, "d128/128x1x64"), (128, 200, "d128/128x2x64"), (256, 200, "d256/64x2x32")):
        q, k, v = (values(rng, (rows, 2, depth), torch.bfloat16) for _ in range(3))
        marks = torch.tensor([0, rows], dtype=torch.int32, device=DEVICE)
        note(f"attention tiles of depth {depth}, {rows} rows")
        operation = hc.Attention(depth ** -0.5)
        check_packed(operation, torch.bfloat16, q, k, v, [0, rows], launch(operation, [q, k, v, marks]))
        assert hc.last_launch_variant() == "attention_tiles/" + want


def test_few_rows_split_their_keys():
    rng = np.random.default_rng(10)
    for rows, shared, keys, want in ((1, 2, 3, "attention_split/d128/16-rows"), (16, 1, 300, "attention_split/d128/16-rows"),
                                     (12, 2, 60, "attention_tiles/d128/128x1x64"), (12, 2, 300, "attention_split/d128/32-rows"),
                                     (16, 4, 200, "attention_tiles/d128/128x2x64"), (16, 4, 1500, "attention_split/d128/64-rows + attention_join/d128/row-to-block")):
        q, k, v = values(rng, (2, rows, 2 * shared, 128), torch.bfloat16, 1.5), values(rng, (2, keys, 2, 128), torch.bfloat16), values(rng, (2, keys, 2, 128), torch.bfloat16)
        lengths = [keys, keys // 3]
        marks = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        note(f"attention of {rows} x {shared} rows over {keys} keys")
        for operation in (hc.Attention(0.088, return_log_sum=True), hc.Attention(0.088, False)):
            check_batched(operation, torch.bfloat16, q, k, v, lengths, launch(operation, [q, k, v, marks]))
            assert hc.last_launch_variant() == want, hc.last_launch_variant()


def test_a_sequence_of_many_steps():
    rng = np.random.default_rng(9)
    q, k, v = values(rng, (1500, 2, 128), torch.bfloat16, 1.5), values(rng, (1500, 1, 128), torch.bfloat16), values(rng, (1500, 1, 128), torch.bfloat16)
    note("attention of 1500 rows")
    for operation in (hc.Attention(0.088, return_log_sum=True), hc.Attention(0.088, True, 333, 200, True), hc.Attention(0.088, False)):
        check_packed(operation, torch.bfloat16, q, k, v, [0, 1500], launch(operation, [q, k, v]))


@pytest.mark.parametrize("tag", ["bf16", "f16"])
@pytest.mark.parametrize("depth", [64, 60])
def test_heads_of_one_projection(tag, depth):
    """Queries, keys and values as views of one packed row, and a batch whose keys are shared by an expanded axis."""
    dtype, rng = TYPES[tag], np.random.default_rng(depth)
    packed = values(rng, (2, 90, 4 + 2 + 2, depth), dtype)
    q, k, v = packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:]
    operation = hc.Attention(depth ** -0.5, True, 0, 0, True)
    note(f"attention of one projection {tag} {depth}")
    check_batched(operation, dtype, q, k, v, None, launch(operation, [q, k, v]))
    shared_k, shared_v = k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1)
    check_batched(operation, dtype, q, shared_k, shared_v, None, launch(operation, [q, shared_k, shared_v]))
    turned = values(rng, (2, 4, 90, depth), dtype)  # heads in front of the rows
    check_batched(operation, dtype, turned.transpose(1, 2), k, v, None, launch(operation, [turned.transpose(1, 2), k, v]))


@pytest.mark.parametrize("tag", ["bf16", "f16", "f32"])
def test_operands_at_any_elements_address(tag):
    dtype, rng = TYPES[tag], np.random.default_rng(7)
    held = [values(rng, (1 + 150 * 2 * 64,), dtype)[1:].view(150, 2, 64) for _ in range(3)]
    operation = hc.Attention(0.125, True, 0, 0, True)
    note(f"attention one element off a boundary {tag}")
    outputs = launch(operation, held)
    check_packed(operation, dtype, *held, [0, 150], outputs)


@pytest.mark.parametrize("tag", ["bf16", "f16"])
@pytest.mark.parametrize("depth,heads", [(64, 2), (128, 1), (256, 1), (80, 1)])
@pytest.mark.parametrize("wrong", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_has_no_part_in_it(tag, depth, heads, wrong):
    """Keys and values that are no numbers: behind a query, before its window, behind the valid keys, in the next sequence."""
    dtype, rng = TYPES[tag], np.random.default_rng(11)
    rows = 210
    q, k, v = (values(rng, (rows, heads, depth), dtype) for _ in range(3))
    for at in (20, 131, 209):
        k[at], v[at, :, ::3] = wrong, wrong
    operation = hc.Attention(depth ** -0.5, True, 40, 2)
    note(f"attention of what is no number {tag} {depth} {wrong}")
    offsets = [0, 100, 210]
    marks = torch.tensor(offsets, dtype=torch.int32, device=DEVICE)
    (out,) = launch(operation, [q, k, v, marks])
    clean_k, clean_v = host(k), host(v)
    seen = np.zeros(rows, bool)
    for a, b in zip(offsets[:-1], offsets[1:]):
        for at in (20, 131, 209):
            if a <= at < b:
                seen[at:min(b, at + 40)] = True
    clean_k[[20, 131, 209]] = 0.0
    clean_v[[20, 131, 209]] = 0.0
    for a, b in zip(offsets[:-1], offsets[1:]):
        want, _, bound, _ = attention_rows(host(q)[a:b], clean_k[a:b], clean_v[a:b], 0, True, 40, 2, operation.scale, dtype)
        rest = ~seen[a:b]
        assert_within(out[a:b][torch.from_numpy(rest).to(DEVICE)], want[rest], bound[rest])
    # padded: behind the valid keys
    q4, k4, v4 = (t[:200].view(2, 100, heads, depth).clone() for t in (q, k, v))
    k4[0, 60:], v4[0, 60:], k4[1, 60:], v4[1, 60:] = wrong, wrong, wrong, wrong
    k4[:, 20:32], v4[:, 20:32] = 0.5, 0.25
    operation = hc.Attention(depth ** -0.5, False)
    outputs = launch(operation, [q4, k4, v4, torch.tensor([60, 50], dtype=torch.int32, device=DEVICE)])
    check_batched(operation, dtype, q4, k4, v4, [60, 50], outputs)


@pytest.mark.parametrize("tag", ["bf16", "f16"])
def test_a_value_that_is_no_number_reaches_the_rows_that_see_it(tag):
    dtype, rng = TYPES[tag], np.random.default_rng(12)
    q, k, v = (values(rng, (150, 1, 64), dtype) for _ in range(3))
    v[70, 0, 5], v[71, 0, 6], v[72, 0, 6] = math.inf, math.nan, 1.0
    operation = hc.Attention(0.125)
    note(f"attention of visible infinities {tag}")
    (out,) = launch(operation, [q, k, v])
    out = out.float().cpu().numpy()[:, 0]
    assert np.isfinite(out[:70]).all() and np.isfinite(out[70:, :5]).all()
    assert (out[70:, 5] == np.inf).all() and np.isnan(out[71:, 6]).all() and np.isfinite(out[70, 6])


@pytest.mark.parametrize("tag", ["bf16", "f16"])
def test_scores_far_apart(tag):
    """A running maximum that grows by much on the way, and one that never does: weights as small as the type has."""
    dtype, rng = TYPES[tag], np.random.default_rng(13)
    q, v = values(rng, (260, 1, 64), dtype), values(rng, (260, 1, 64), dtype)
    for slope in (0.05, -0.05):
        k = (q.float().mean(0, keepdim=True) + 0.1 * torch.from_numpy(rng.normal(0, 1, (260, 1, 64)).astype(np.float32)).to(DEVICE))
        k = (k + torch.arange(260, device=DEVICE)[:, None, None] * slope * torch.sign(q.float().mean(0, keepdim=True))).to(dtype)
        operation = hc.Attention(1.0, False, 0, 0, True)
        note(f"attention of scores far apart {tag} {slope}")
        check_packed(operation, dtype, q, k, v, [0, 260], launch(operation, [q, k, v]))


def test_more_keys_than_32_bit_offsets_reach():
    """Rows that lie further than 4 GiB apart: what is read is the row's own."""
    rng, rows, gap = np.random.default_rng(14), 40, 2 ** 27 - 8
    free = torch.cuda.mem_get_info()[0]
    if free < 3 * rows * gap:
        pytest.skip("needs memory for operands of some GiB")
    note("attention over rows of 128 MiB")
    held = torch.zeros(rows * gap // 2, dtype=torch.bfloat16, device=DEVICE)
    k = held.as_strided((rows, 1, 64), (gap // 2, 64, 1))
    k.copy_(values(rng, (rows, 1, 64), torch.bfloat16))
    q, v = values(rng, (rows, 2, 64), torch.bfloat16), values(rng, (rows, 1, 64), torch.bfloat16)
    operation = hc.Attention(0.125)
    check_packed(operation, torch.bfloat16, q, k, v, [0, rows], launch(operation, [q, k, v]))
    check_packed(operation, torch.bfloat16, q, v, k, [0, rows], launch(operation, [q, v, k]))


def test_outputs_that_overlap_an_operand_are_refused():
    rng = np.random.default_rng(15)
    q, k, v = (values(rng, (40, 2, 64), torch.bfloat16) for _ in range(3))
    bound = tio.Bound(context(), hc.Attention(0.125, return_log_sum=True), [tio.desc_of(t) for t in (q, k, v)])
    out, logs = bound.outputs()
    note("attention into its own operands")
    for inputs, outputs in (([q, k, v], [q, logs]), ([q, k, v], [v, logs]), ([out.view(-1)[:40 * 128].view(40, 2, 64), k, v], [out, logs]),
                            ([q, k, v], [out, out.view(-1)[:160].view(torch.float32).view(40, 2)])):
        with pytest.raises(hc.StatusError) as refused:
            bound.submit(inputs, outputs)
        assert refused.value.is_invalid_argument()


def test_results_are_the_same_bits_every_time_and_on_any_stream():
    rng = np.random.default_rng(16)
    q, k, v = values(rng, (700, 8, 128), torch.bfloat16), values(rng, (700, 2, 128), torch.bfloat16), values(rng, (700, 2, 128), torch.bfloat16)
    bound = tio.Bound(context(), hc.Attention(0.088, True, 0, 0, True), [tio.desc_of(t) for t in (q, k, v)])
    note("attention twice, and on another stream")
    first, second, third = bound.outputs(), bound.outputs(), bound.outputs()
    bound.submit([q, k, v], first)
    bound.submit([q, k, v], second)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        bound.submit([q, k, v], third)
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)
