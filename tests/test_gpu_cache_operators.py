"""Caches of 4 bits, RotaryAppend, PageBounds, PagedSelect and PagedAttention over pages of each key head, against their
definitions in 64 bits, one by one and as a decoding step runs them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyle_amd import compute as hc
from hyle_amd import torch_io as tio

import cache_support as cs
from attention_support import assert_within, attention_rows
from gpu_support import DEVICE, context, note

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "mx4": torch.uint8}
HALF, PAIRS = hc.RopeLayout.kHalfSplit, hc.RopeLayout.kInterleaved


def device(array):
    return torch.from_numpy(np.ascontiguousarray(array)).to(DEVICE)


def values(rng, shape, tag, std=1.0):
    x = device(rng.normal(0, std, shape).astype(np.float32))
    return x.to(torch.bfloat16).to(TYPES[tag]) if tag == "e4m3" else x.to(TYPES[tag])


def host(tensor):
    return tensor.float().cpu().double().numpy()


def cache_of(rng, pages, heads, page, depth, tag):
    if tag != "mx4":
        return values(rng, (pages, 2, heads, page, depth), tag)
    codes = rng.integers(0, 256, (pages, 2, heads, page, depth // 2)).astype(np.uint8)
    scales = rng.integers(124, 129, (pages, 2, heads, page, depth // 32)).astype(np.uint8)
    return device(cs.mx4_join(codes, scales))


def off_by(tensor, size):
    """The same values at an address `size` bytes past a whole vector's."""
    raw = torch.empty(tensor.numel() * tensor.element_size() + size, dtype=torch.uint8, device=DEVICE)[size:]
    return raw.copy_(tensor.contiguous().view(torch.uint8).view(-1)).view(tensor.dtype).view(tensor.shape)


def submit(operation, inputs, outputs=None):
    bound = tio.Bound(context(), operation, [tio.desc_of(t) for t in inputs])
    made = bound.outputs()
    if outputs is not None:
        made[:len(outputs)] = outputs
    bound.submit(inputs, made)
    torch.cuda.synchronize()
    return made


def pages_of(rng, lengths, page, spare=2, columns=None):
    """A table whose pages are in no order, and how many pages there are."""
    held = [-(-max(0, n) // page) for n in lengths]
    order, columns, at = rng.permutation(sum(held) + spare).astype(np.int32), columns or max(held + [1]), 0
    table = np.full((len(lengths), columns), -1, np.int32)
    for row, count in zip(table, held):
        row[:count] = order[at:at + count][:columns]
        at += count
    return table, sum(held) + spare


# ---- 4 bits ---------------------------------------------------------------------------------
def hard_rows(rng, tokens, heads, depth, dtype):
    """Rows with blocks of every kind: ties, ends of the exponent's range, zeros of both signs, what is no number."""
    x = rng.normal(0, 1, (tokens, heads, depth)) * np.exp2(rng.integers(-12, 12, (tokens, heads, 1)))
    blocks = x.reshape(-1, 32)
    kinds = [np.zeros(32), -np.zeros(32), np.tile([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], 4), np.tile([7.0, -0.25, 1.0, -5.0], 8),
             np.tile([7.0078125, 0.5, 1.5, -2.5], 8), np.full(32, np.finfo(np.float32).max if dtype != torch.float16 else 65504.0),
             np.full(32, 2.0 ** -126), np.full(32, 2.0 ** -133), np.where(np.arange(32) == 7, np.nan, 1.0), np.where(np.arange(32) == 31, np.inf, 1.0)]
    for i, kind in enumerate(kinds[:len(blocks)]):
        blocks[(i * 7) % len(blocks)] = kind
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


@pytest.mark.parametrize("tag", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("depth,page,tokens,off", [(128, 16, 40, 0), (32, 1, 9, 0), (96, 7, 130, 0), (64, 24, 50, 3), (256, 64, 300, 0), (160, 16, 33, 1)])
def test_rows_are_kept_in_four_bits(tag, depth, page, tokens, off):
    rng, heads, pages = np.random.default_rng(depth + tokens), 3, -(-tokens // page) + 2
    dtype = TYPES[tag]
    keys, vals = hard_rows(rng, tokens, heads, depth, dtype), hard_rows(rng, tokens, heads, depth, dtype).flip(0)
    cache = cache_of(rng, pages, heads, page, depth, "mx4")
    cache = off_by(cache, off) if off else cache
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    slots[2::9] = rng.choice([-1, pages * page, 2 ** 31 - 1, -2 ** 31], len(slots[2::9]))
    want = cache.cpu().numpy().copy()
    codes, scales = cs.mx4_split(want)
    for side, rows in ((0, keys), (1, vals)):
        row_codes, row_scales = cs.mx4_encode(rows.double().numpy(), dtype)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page:
                codes[slot // page, side, :, slot % page] = row_codes[t]
                scales[slot // page, side, :, slot % page] = row_scales[t]
    note(f"append in 4 bits {tag} depth {depth} page {page} tokens {tokens} off {off}")
    (got,) = submit(hc.PagedAppend(pages, page, hc.DataType.kUInt8), [keys.to(DEVICE), vals.to(DEVICE), device(slots)], [cache])
    got = got.cpu().numpy()
    got_codes, got_scales = cs.mx4_split(got)
    assert np.array_equal(got_scales, scales)
    numbers = np.repeat(scales != 255, 16, axis=-1)  # (codes of a block that is no number are any)
    assert np.array_equal(got_codes[numbers], codes[numbers])


@pytest.mark.parametrize("tag", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("depth", [256, 224])
def test_every_code_of_every_scale_is_read(tag, depth):
    """One key: its weight is 1, so the output is the value, rounded to the queries' type."""
    blocks = depth // 32
    pages = -(-256 // blocks)
    scales = (np.arange(pages * blocks) % 256).astype(np.uint8).reshape(pages, 1, 1, blocks)
    codes = np.broadcast_to(np.tile(np.arange(16, dtype=np.uint8), depth // 16), (pages, 1, 1, depth))
    packed = codes[..., 0::2] | codes[..., 1::2] << 4
    side = cs.mx4_join(packed, scales)
    cache = device(np.stack((np.zeros_like(side), side), axis=1))
    note(f"every code of every scale {tag} depth {depth}")
    (got,) = submit(hc.PagedAttention(), [torch.zeros((pages, 2, depth), dtype=TYPES[tag], device=DEVICE), cache,
                                          torch.arange(pages, dtype=torch.int32, device=DEVICE)[:, None], torch.ones(pages, dtype=torch.int32, device=DEVICE)])
    with np.errstate(over="ignore"):
        want = torch.from_numpy(cs.mx4_decode(packed, scales).astype(np.float32)[:, 0]).to(TYPES[tag]).double().numpy()
    got = host(got)
    # (f32's subnormal numbers, of bf16 and f32 alike, may come out as zeros of the matrix unit and of exponentials' products)
    want = np.broadcast_to(want, got.shape)
    tiny = np.abs(want) < 2.0 ** -126
    assert np.array_equal(got[~tiny], want[~tiny], equal_nan=True)
    assert (np.abs(got[tiny]) <= np.abs(want[tiny])).all()


# type, depth, query heads, key heads, page, lengths, new tokens, window, sinks, logarithms, bytes off a vector
DECODES_4 = [
    ("bf16", 128, 32, 8, 16, (1, 700, 33, 0, 128, 129, 2500), 1, 0, 0, True, 0),
    ("f16", 96, 20, 5, 32, (500, 3001, 4, 2), 4, 256, 4, True, 0),
    ("bf16", 256, 16, 2, 16, (9001,), 1, 0, 0, True, 0),
    ("f16", 64, 8, 8, 8, (77, 1, 640), 2, 0, 0, False, 0),
    ("bf16", 32, 6, 1, 1, (300, 17), 3, 0, 0, False, 0),
    ("f16", 224, 12, 2, 24, (1000, 31), 5, 90, 0, True, 0),
    ("bf16", 128, 40, 5, 256, (1500, 255, 256, 257), 8, 0, 0, False, 0),
    ("bf16", 160, 4, 4, 7, (91, 800), 1, 64, 16, True, 0),
    ("f32", 96, 6, 3, 16, (70, 1, 0), 2, 30, 3, True, 0),
    ("bf16", 128, 4, 2, 16, (300, 40), 2, 0, 0, True, 1),
    ("f16", 64, 4, 2, 16, (300, 40), 1, 100, 0, True, 2),
    ("f16", 64, 40, 1, 16, (300, 40), 2, 0, 0, True, 4),
    # up to 16, 32 and 64 rows of a key head, of every depth's kernel
    ("bf16", 32, 4, 2, 16, (300, 700), 3, 0, 0, False, 0), ("f16", 32, 9, 1, 16, (300, 1, 700), 3, 100, 7, True, 0),
    ("bf16", 32, 14, 2, 16, (140, 1000), 8, 0, 0, False, 0), ("f16", 64, 24, 1, 16, (140, 1000), 1, 0, 0, True, 0),
    ("bf16", 96, 24, 2, 8, (140, 3, 1000), 2, 0, 0, True, 0), ("f16", 96, 40, 1, 8, (140, 1000), 1, 0, 0, False, 0),
    ("f16", 128, 8, 1, 4, (5, 1000), 4, 64, 0, True, 0), ("bf16", 224, 4, 2, 16, (900, 70), 1, 0, 0, True, 0),
    ("bf16", 128, 8, 2, 16, (0, -3, 0), 1, 0, 0, True, 0), ("f16", 64, 8, 2, 16, (0,), 2, 0, 0, True, 0),
    ("f16", 192, 20, 1, 16, (900, 70), 3, 0, 0, False, 0), ("bf16", 256, 8, 1, 16, (900, 70, 2), 3, 0, 0, True, 0),
]


@pytest.mark.parametrize("tag,depth,queries,heads,page,lengths,new,window,sinks,logs,off", DECODES_4)
def test_attention_over_four_bits(tag, depth, queries, heads, page, lengths, new, window, sinks, logs, off):
    rng = np.random.default_rng(depth + queries)
    table, pages = pages_of(rng, lengths, page, columns=max(40, -(-max(lengths) // page)))
    cache = cache_of(rng, pages, heads, page, depth, "mx4")
    cache = off_by(cache, off) if off else cache
    query = values(rng, (len(lengths), new, queries, depth), tag, 0.7)
    operation = hc.PagedAttention(depth ** -0.5, window, sinks, logs)
    note(f"attention over 4 bits {tag} depth {depth} heads {queries}/{heads} page {page} lengths {lengths} new {new} window {window} off {off}")
    outputs = submit(operation, [query, cache, device(table), torch.tensor(lengths, dtype=torch.int32, device=DEVICE)])
    held = cs.cache_values(cache)
    for i, n in enumerate(lengths):
        place = np.arange(max(n, 0))
        k, v = (held[table[i, place // page], side, :, place % page] for side in (0, 1))
        want, want_logs, bound, log_bound = attention_rows(host(query[i]), k, v, max(n, 0) - new, True, window, sinks, operation.scale, query.dtype)
        assert_within(outputs[0][i], want, bound)
        if logs:
            assert_within(outputs[1][i], want_logs, log_bound)


@pytest.mark.parametrize("tag,queries,depth", [("bf16", 8, 128), ("f16", 48, 64), ("f32", 8, 64)])
def test_values_of_keys_that_a_row_does_not_see_count_for_nothing(tag, queries, depth):
    """The last of three new tokens is NaN, or beyond the type: the rows before it are as they are without."""
    rng, lengths, new, page = np.random.default_rng(9), (200, 131, 3), 3, 16
    table, pages = pages_of(rng, lengths, page)
    cache = cache_of(rng, pages, 2, page, depth, "mx4")
    raw = cache.cpu().numpy()
    scales = cs.mx4_split(raw)[1]
    for i, n in enumerate(lengths):
        scales[table[i, (n - 1) // page], 1, :, (n - 1) % page] = (255, 254, 255)[i]
    query = values(rng, (3, new, queries, depth), tag)
    note(f"values that are no numbers in 4 bits {tag} depth {depth}")
    (got,) = submit(hc.PagedAttention(0.1), [query, device(raw), device(table), torch.tensor(lengths, dtype=torch.int32, device=DEVICE)])
    held = cs.cache_values(device(raw))
    for i, n in enumerate(lengths):
        place = np.arange(n)
        k, v = (held[table[i, place // page], side, :, place % page] for side in (0, 1))
        want, _, bound, _ = attention_rows(host(query[i])[:2], k[:-1], v[:-1], n - new, True, 0, 0, 0.1, query.dtype)
        assert_within(got[i, :2], want, bound)
    assert torch.isnan(got[0, 2]).all() and torch.isnan(got[2, 2]).all()


# ---- pages of each key head ------------------------------------------------------------------
@pytest.mark.parametrize("tag,cache_tag,depth,queries,heads,page,new,logs,off", [
    ("bf16", "bf16", 128, 32, 8, 16, 1, False, 0), ("f16", "mx4", 128, 20, 5, 32, 3, True, 0), ("bf16", "e4m3", 64, 12, 3, 8, 2, True, 0),
    ("f16", "f16", 80, 10, 5, 16, 8, True, 0), ("bf16", "mx4", 256, 34, 2, 16, 2, False, 0), ("bf16", "bf16", 128, 3, 1, 16, 2, True, 0),
    ("f32", "f32", 40, 6, 3, 5, 2, True, 0), ("bf16", "bf16", 72, 6, 3, 16, 1, True, 2), ("f32", "mx4", 32, 8, 4, 16, 1, True, 0)])
def test_attention_over_pages_of_each_key_head(tag, cache_tag, depth, queries, heads, page, new, logs, off):
    rng, sequences, columns, shared = np.random.default_rng(depth + new), 4, 40, queries // heads
    pages = 120
    cache = cache_of(rng, pages, heads, page, depth, cache_tag)
    cache = off_by(cache, off) if off else cache
    table = rng.integers(0, pages, (sequences, heads, columns)).astype(np.int32)  # any page, also twice
    table[1, 0, 3] = -1
    lengths = rng.integers(new, columns * page + 1, (sequences, heads)).astype(np.int32)
    lengths[0, 0], lengths[2, heads - 1], lengths[3, 0] = columns * page, 0, 1
    query = values(rng, (sequences, new, queries, depth), tag)
    note(f"pages of key heads {tag} {cache_tag} depth {depth} heads {queries}/{heads} page {page} new {new}")
    outputs = submit(hc.PagedAttention(0.11, return_log_sum=logs), [query, cache, device(table), device(lengths)])
    held = cs.cache_values(cache)
    for i in range(sequences):
        for h in range(heads):
            n = int(lengths[i, h])
            place, mine = np.arange(n), slice(h * shared, (h + 1) * shared)
            k, v = (held[table[i, h, place // page], side, h, place % page][:, None] for side in (0, 1))
            gone = np.flatnonzero(table[i, h, place // page] < 0)
            want, want_logs, bound, log_bound = attention_rows(host(query[i])[:, mine], k, v, n - new, True, 0, 0, 0.11, query.dtype, gone)
            assert_within(outputs[0][i, :, mine], want, bound)
            if logs:
                assert_within(outputs[1][i, :, mine], want_logs, log_bound)


# ---- RotaryAppend ----------------------------------------------------------------------------
# type, cache, queries, heads, depth, rotary, layout, page, tokens, wide positions, frequencies of each token, bytes off a vector
ROTARIES = [
    ("bf16", "bf16", 32, 8, 128, 128, HALF, 16, 64, False, False, 0),
    ("bf16", "e4m3", 8, 2, 128, 128, HALF, 64, 300, False, False, 0),
    ("f16", "mx4", 20, 5, 96, 64, PAIRS, 16, 130, False, False, 0),
    ("f16", "f16", 4, 4, 64, 32, HALF, 8, 1, True, False, 0),
    ("bf16", "mx4", 6, 2, 256, 256, HALF, 32, 77, False, True, 0),
    ("f32", "f32", 3, 3, 80, 80, PAIRS, 5, 41, True, True, 0),
    ("f32", "mx4", 2, 1, 32, 16, HALF, 16, 19, False, False, 0),
    ("f32", "e4m3", 2, 2, 24, 24, PAIRS, 16, 19, False, False, 0),
    ("bf16", "bf16", 0, 3, 72, 40, HALF, 16, 33, False, False, 0),
    ("f16", "e4m3", 0, 2, 128, 64, PAIRS, 16, 33, False, False, 0),
    ("bf16", "bf16", 5, 1, 63, 30, PAIRS, 7, 50, False, False, 0),
    ("f16", "f16", 5, 1, 66, 66, HALF, 7, 50, False, False, 0),
    ("bf16", "bf16", 4, 2, 128, 128, HALF, 16, 21, False, False, 2),
    ("bf16", "e4m3", 4, 2, 128, 128, HALF, 16, 21, False, False, 2),
    ("f16", "mx4", 4, 2, 64, 64, PAIRS, 16, 21, False, False, 2),
    ("bf16", "bf16", 1, 1, 1024, 512, HALF, 16, 9, False, False, 0),
    ("bf16", "bf16", 4, 2, 2, 2, HALF, 16, 9, False, False, 0),
    ("bf16", "bf16", 4, 2, 128, 2, PAIRS, 16, 65, False, False, 0),
    ("f16", "f16", 4, 2, 128, 120, PAIRS, 16, 65, False, False, 0),
    ("bf16", "mx4", 4, 2, 128, 120, HALF, 16, 65, False, False, 0),
    ("bf16", "bf16", 7, 3, 128, 64, HALF, 16, 1, False, False, 0), ("f16", "f16", 6, 2, 80, 80, PAIRS, 16, 333, False, True, 0),
    ("f16", "e4m3", 6, 2, 96, 48, HALF, 16, 333, True, False, 0), ("bf16", "e4m3", 5, 1, 256, 16, PAIRS, 8, 70, False, False, 0),
    ("bf16", "mx4", 32, 8, 128, 128, HALF, 16, 64, False, False, 0), ("f16", "mx4", 3, 3, 32, 32, HALF, 16, 4500, False, False, 0),
    ("bf16", "mx4", 2, 1, 992, 960, PAIRS, 4, 5, False, False, 0), ("f32", "f32", 4, 2, 64, 32, HALF, 16, 40, False, False, 0),
    ("f32", "e4m3", 4, 2, 64, 64, PAIRS, 16, 40, False, False, 0), ("bf16", "bf16", 2, 1, 16, 16, HALF, 16, 5000, False, False, 0),
    ("bf16", "mx4", 6, 2, 64, 64, HALF, 1, 40, False, False, 0), ("bf16", "mx4", 6, 2, 64, 64, HALF, 16, 40, False, False, 4),
]


@pytest.mark.parametrize("tag,cache_tag,queries,heads,depth,rotary,layout,page,tokens,wide,stepped,off", ROTARIES)
def test_rows_are_rotated_on_the_way(tag, cache_tag, queries, heads, depth, rotary, layout, page, tokens, wide, stepped, off):
    """Bit by bit: every rounding of the definition is one of the kernel's."""
    rng, rows, pages = np.random.default_rng(depth + tokens + queries), queries + 2 * heads, -(-tokens // page) + 2
    projected = values(rng, (tokens, rows, depth), tag, 2.0)
    projected = off_by(projected, off) if off else projected
    positions = rng.integers(-40, 140000, tokens).astype(np.int64 if wide else np.int32)
    positions[0], positions[-1] = 0, 3 * 10 ** 7
    if wide:
        positions[-1] = 5 * 10 ** 12
    frequencies = (10000.0 ** (-2 * np.arange(rotary // 2) / rotary)).astype(np.float32)
    if stepped:
        frequencies = frequencies * rng.uniform(0.5, 1.5, (tokens, 1)).astype(np.float32)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    slots[3::7] = rng.choice([-1, pages * page, 2 ** 31 - 1, -2 ** 31], len(slots[3::7]))
    cache = cache_of(rng, pages, heads, page, depth, cache_tag)
    before = cache.clone()
    note(f"rotary append {tag} -> {cache_tag} heads {queries}/{heads} depth {depth}/{rotary} {layout.name} page {page} tokens {tokens} off {off}")
    outputs = submit(hc.RotaryAppend(pages, page, tio.desc_of(cache).data_type, heads, layout),
                     [projected, device(positions), device(frequencies), device(slots)], [cache])
    x = projected.float().cpu().numpy()
    turned = np.concatenate((cs.rotated(x[:, :queries + heads], positions, frequencies, layout == HALF), x[:, queries + heads:]), axis=1)
    if queries:
        assert torch.equal(outputs[1].cpu(), torch.from_numpy(turned[:, :queries]).to(TYPES[tag]))
    kept = (slots >= 0) & (slots < pages * page)
    at, place = slots[kept] // page, slots[kept] % page
    new = turned[kept, queries:].reshape(-1, 2, heads, depth)
    if cache_tag == "mx4":
        want = before.cpu().numpy()
        codes, scales = cs.mx4_split(want)
        row_codes, row_scales = cs.mx4_encode(new.astype(np.float64), TYPES[tag])
        for side in (0, 1):
            codes[at, side, :, place], scales[at, side, :, place] = row_codes[:, side], row_scales[:, side]
        assert np.array_equal(cache.cpu().numpy(), want)
        return
    rounded = torch.from_numpy(new).clamp(-448, 448).to(torch.float8_e4m3fn) if cache_tag == "e4m3" else torch.from_numpy(new).to(TYPES[tag])
    want, rounded = before.cpu().view(torch.uint8).view(pages, 2, heads, page, -1), rounded.view(torch.uint8).view(*new.shape[:3], -1)
    for side in (0, 1):
        want[torch.from_numpy(at).long(), side, :, torch.from_numpy(place).long()] = rounded[:, side]
    assert torch.equal(cache.cpu().view(torch.uint8).view(want.shape), want)


@pytest.mark.parametrize("cache_tag", ["bf16", "mx4"])
def test_rotary_append_of_strided_rows(cache_tag):
    """Rows within a wider projection, heads apart, and one row for all tokens; what is only stored keeps its bits."""
    rng = np.random.default_rng(2)
    wide = values(rng, (30, 9, 160), "bf16")
    frequencies = device((10.0 ** -np.arange(32)).astype(np.float32))
    positions, slots = torch.arange(30, dtype=torch.int32, device=DEVICE), torch.randperm(48, device=DEVICE)[:30].to(torch.int32)
    for projected in (wide[:, 1:, 32:96], wide[:, ::2, :64][:, :4], wide[:1, :8, :64].expand(30, -1, -1), wide.transpose(0, 1)[:, 1:7, 8:72].transpose(0, 1)[:6, :8]):
        heads, tokens = 2, projected.shape[0]
        caches = [cache_of(np.random.default_rng(3), 3, heads, 16, 64, cache_tag) for _ in range(2)]
        operation = hc.RotaryAppend(3, 16, tio.desc_of(caches[0]).data_type, heads, HALF)
        note(f"rotary append of strides {projected.stride()}")
        got = submit(operation, [projected, positions[:tokens], frequencies, slots[:tokens]], caches[:1])
        want = submit(operation, [projected.contiguous(), positions[:tokens], frequencies, slots[:tokens]], caches[1:])
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    odd = torch.full((4, 4, 64), float("nan"), dtype=torch.bfloat16, device=DEVICE)
    odd.view(torch.int16)[:, 3] = 0x7F81 + torch.arange(64, dtype=torch.int16, device=DEVICE)
    cache = torch.zeros((1, 2, 1, 4, 64), dtype=torch.bfloat16, device=DEVICE)
    submit(hc.RotaryAppend(1, 4, hc.DataType.kBFloat16, 1, HALF), [odd, positions[:4], frequencies, positions[:4]], [cache])
    assert torch.equal(cache.view(torch.int16)[0, 1, 0], odd.view(torch.int16)[:, 3]) and torch.isnan(cache[0, 0]).all()


def test_rotary_append_is_rope_and_paged_append():
    """Beside the two operations that it joins: both round once (2^-8 each, of values that are a rounding larger at most), and cos and sin
    of RoPE are f32 functions (2^-21 of the pair's length covers theirs and the products')."""
    rng, tokens = np.random.default_rng(6), 70
    projected = values(rng, (tokens, 12, 128), "bf16")
    positions, slots = torch.arange(5, 5 + tokens, dtype=torch.int32, device=DEVICE), torch.arange(tokens, dtype=torch.int32, device=DEVICE)
    frequencies = device((10000.0 ** (-np.arange(64) / 64)).astype(np.float32))
    cache = torch.zeros((5, 2, 2, 16, 128), dtype=torch.bfloat16, device=DEVICE)
    joined, other = cache.clone(), cache.clone()
    note("rotary append beside rope and paged append")
    got = submit(hc.RotaryAppend(5, 16, hc.DataType.kBFloat16, 2, HALF), [projected, positions, frequencies, slots], [joined])
    (query,) = submit(hc.RoPE(128, 0, HALF), [projected[:, :8].contiguous(), positions, frequencies])
    (key,) = submit(hc.RoPE(128, 0, HALF), [projected[:, 8:10].contiguous(), positions, frequencies])
    submit(hc.PagedAppend(5, 16, hc.DataType.kBFloat16), [key, projected[:, 10:], slots], [other])
    size = projected.float().view(tokens, 12, 2, 64).norm(dim=2).repeat(1, 1, 2)
    for a, b, most in ((got[1], query, size[:, :8]), (joined[:, 0].transpose(1, 2).reshape(80, 2, 128)[:tokens], key, size[:, 8:10])):
        assert ((a.float() - b.float()).abs() <= 1.01 * 2.0 ** -7 * b.float().abs() + 2.0 ** -21 * most).all()
    assert torch.equal(joined[:, 1], other[:, 1])


# ---- PageBounds ------------------------------------------------------------------------------
@pytest.mark.parametrize("cache_tag", ["bf16", "f16", "f32", "e4m3", "mx4"])
@pytest.mark.parametrize("depth,heads,page,newest,off", [(128, 8, 16, 1, 0), (64, 3, 1, 0, 0), (96, 2, 24, 30, 0), (256, 1, 256, 0, 0), (32, 5, 7, 4, 0),
                                                         (128, 2, 64, 0, 4), (64, 2, 16, 0, 2), (320, 2, 16, 500, 0),
                                                         (64, 1, 1100, 0, 0), (128, 2, 600, 700, 0), (160, 1, 288, 0, 0), (72, 3, 16, 2, 0), (256, 2, 8, 0, 0)])
def test_bounds_of_pages(cache_tag, depth, heads, page, newest, off):
    if cache_tag == "mx4" and depth % 32 != 0:
        pytest.skip("4 bits come in blocks of 32")
    rng, lengths = np.random.default_rng(depth + page), (1, 300, page, 0, 3 * page + 1, -5)
    table, pages = pages_of(rng, lengths, page)
    table[1, 0] = (-1, pages, 2 ** 31 - 1)[heads % 3]
    cache = cache_of(rng, pages, heads, page, depth, cache_tag)
    if cache_tag == "mx4":
        raw = cache.cpu().numpy()
        scales = cs.mx4_split(raw)[1]
        scales.reshape(-1)[::37] = 255
        scales.reshape(-1)[1::53] = 0
        scales.reshape(-1)[2::59] = 254
        cache = device(raw)
    else:
        flat = cache.view(-1)
        for step, odd in ((101, float("nan")), (211, 0.0), (307, -0.0)) + (() if cache_tag == "e4m3" else ((401, float("inf")), (503, float("-inf")))):
            flat[::step] = torch.tensor(odd).to(flat.dtype)
        if cache_tag == "f32":
            flat[3::97] = 3.4e38
            flat[5::89] = -1e-40
        if cache_tag == "bf16":  # (a signaling one)
            cache.view(torch.int16).view(-1)[11::113] = 0x7F81
    cache[int(table[4, 0]), 0, 0].view(torch.uint8)[...] = 255  # channels without a number (of e4m3, f16, bf16, f32 and 4 bits)
    before = rng.integers(0, 2 ** 15, (pages, 2, heads, depth)).astype(np.uint16)
    bounds = device(before.view(np.int16)).view(torch.bfloat16)
    held = off_by(cache, off) if off and off % cache.element_size() == 0 else cache
    note(f"bounds {cache_tag} depth {depth} heads {heads} page {page} newest {newest} off {off}")
    submit(hc.PageBounds(newest), [held, device(table), torch.tensor(lengths, dtype=torch.int32, device=DEVICE)], [bounds])
    with np.errstate(over="ignore"):
        values_ = cs.cache_values(cache).astype(np.float32)
    want = cs.page_bounds(values_, table, lengths, newest, before)
    got = bounds.view(torch.int16).cpu().numpy().view(np.uint16)
    same = (got == want) | (((got | want) & 0x7FFF) == 0)  # (zeros of either sign)
    assert same.all(), np.argwhere(~same)[:3]


def test_bounds_of_a_cache_within_another():
    """Pages and heads of a larger cache by their strides."""
    rng = np.random.default_rng(12)
    whole = values(rng, (20, 2, 6, 16, 192), "bf16")
    part = whole[3:17:2, :, 1:5, :, 64:]
    table, lengths = device(np.array([[0, 3, 6], [5, 1, 2]], np.int32)), torch.tensor([40, 48], dtype=torch.int32, device=DEVICE)
    note("bounds of a part of a cache")
    got, want = (submit(hc.PageBounds(), [cache, table, lengths], [torch.zeros((7, 2, 4, 128), dtype=torch.bfloat16, device=DEVICE)])[0]
                 for cache in (part, part.contiguous()))
    assert torch.equal(got, want) and (want[[0, 1, 2, 3, 5, 6]] != 0).any(-1).all() and (want[4] == 0).all()


# ---- PagedSelect -----------------------------------------------------------------------------
def bounds_of(rng, pages, heads, depth):
    center, width = rng.normal(0, 0.5, (pages, heads, depth)), np.abs(rng.normal(0, 0.4, (pages, heads, depth))) + 1.0
    return device(np.stack((center - width, center + width), axis=1).astype(np.float32)).to(torch.bfloat16)


# type, queries, heads, depth, page, count, new, lengths, bytes off a vector
SELECTS = [
    ("bf16", 32, 8, 128, 16, 20, 1, (1000, 40, 1, 0, 3000), 0),
    ("f16", 16, 2, 256, 32, 60, 2, (9000,), 0),
    ("bf16", 5, 5, 64, 8, 5, 3, (300, 2, 39, 41), 0),
    ("f32", 6, 2, 80, 16, 3, 1, (200, 33, 49), 0),
    ("f16", 12, 3, 96, 1, 12, 8, (100, 13, 12, 11, 5), 0),
    ("bf16", 8, 1, 33, 16, 300, 4, (7000, 4801), 0),
    ("bf16", 3, 3, 7, 2, 1100, 1, (6000,), 0),
    ("bf16", 8, 2, 128, 16, 9, 1, (300, 2000), 2),
    ("f16", 24, 3, 128, 16, 17, 5, (300, 2000, 4), 0),
    ("bf16", 64, 1, 128, 64, 4, 8, (5000, 640), 0),
    # two and four waves to the query rows, rows that no group of four fills, few and many pages of every depth's kernel, blocks that end inside
    # a sequence, pages that threads keep in registers and those that they do not
    ("f16", 7, 1, 64, 16, 9, 1, (3000, 170), 0), ("bf16", 14, 2, 256, 16, 9, 1, (3000, 170), 0), ("f32", 12, 2, 128, 16, 9, 2, (3000, 170), 0),
    ("bf16", 6, 3, 64, 1, 700, 2, (30011, 29000), 0), ("f16", 5, 1, 128, 1, 30, 3, (40001,), 0), ("bf16", 4, 2, 256, 1, 3000, 1, (9000, 4099, 300), 0),
    ("f32", 2, 2, 136, 1, 5, 1, (16384, 16385), 0), ("f16", 4, 1, 96, 1, 16000, 1, (17000, 40000), 0),
    ("bf16", 24, 2, 64, 16, 9, 1, (3000, 170), 0),
]


@pytest.mark.parametrize("tag,queries,heads,depth,page,count,new,lengths,off", SELECTS)
def test_the_best_pages_are_chosen(tag, queries, heads, depth, page, count, new, lengths, off):
    rng = np.random.default_rng(depth + count)
    table, pages = pages_of(rng, lengths, page)
    bounds = bounds_of(rng, pages, heads, depth)
    bounds = off_by(bounds, off) if off else bounds
    query = values(rng, (len(lengths), new, queries, depth), tag)
    note(f"select {tag} heads {queries}/{heads} depth {depth} page {page} count {count} new {new} lengths {lengths} off {off}")
    got = submit(hc.PagedSelect(count, page), [query, bounds, device(table), torch.tensor(lengths, dtype=torch.int32, device=DEVICE)])
    want = cs.selected(host(query), host(bounds), table, lengths, heads, page, count)
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])


def test_choices_at_the_edges():
    """Equal scores, scores that are no numbers or infinite, pages that are not there, lengths beyond the table."""
    rng, page, heads, depth, lengths = np.random.default_rng(1), 16, 4, 64, (900, 900, 900, 2 ** 31 - 1, -3)
    table, pages = pages_of(rng, (900, 900, 900, 900, 0), page, columns=57)
    bounds = bounds_of(rng, pages, heads, depth)
    bounds[table[0].astype(np.int64)] = bounds[int(table[0, 0])].clone()       # equal scores
    bounds[int(table[1, 9]), 1, 0, 5] = float("nan")
    bounds[int(table[1, 7]), 1, 1] = float("inf")
    bounds[int(table[1, 8]), 0, 1] = float("-inf")                             # inf - inf with queries of both signs: none
    bounds[int(table[1, 11]), :, 2] = torch.tensor([float("inf"), float("-inf")], dtype=torch.bfloat16, device=DEVICE)[:, None]
    table[2, 4:50:3] = -1
    table[2, 5:50:5] = pages
    query = values(rng, (5, 1, 8, depth), "bf16")
    query[2, :, 6] = 0.0
    query[3, :, 2] = float("nan")
    note("select at the edges")
    for count in (3, 8, 31, 56, 57):
        got = submit(hc.PagedSelect(count, page), [query[:, 0], bounds, device(table), torch.tensor(lengths, dtype=torch.int32, device=DEVICE)])
        with np.errstate(invalid="ignore"):
            want = cs.selected(host(query), host(bounds), table, lengths, heads, page, count)
        assert np.array_equal(got[0].cpu().numpy(), want[0]), count
        assert np.array_equal(got[1].cpu().numpy(), want[1]), count


def test_a_choice_where_no_page_has_bounds():
    """A cache without pages: all scores are the least, so the earlier pages of the table are chosen."""
    rng, lengths = np.random.default_rng(3), (700, 40)
    table, _ = pages_of(rng, lengths, 16)
    query = values(rng, (2, 1, 4, 64), "bf16")
    bounds = torch.zeros((0, 2, 2, 64), dtype=torch.bfloat16, device=DEVICE)
    note("select without pages")
    got = submit(hc.PagedSelect(5, 16), [query, bounds, device(table), torch.tensor(lengths, dtype=torch.int32, device=DEVICE)])
    want = cs.selected(host(query), np.zeros((0, 2, 2, 64)), table, lengths, 2, 16, 5)
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])


# ---- together --------------------------------------------------------------------------------
@pytest.mark.parametrize("tag,cache_tag", [("bf16", "bf16"), ("f16", "mx4"), ("bf16", "e4m3")])
def test_steps_of_sparse_decoding(tag, cache_tag):
    """New tokens into the cache, their pages' bounds, the choice, the attention over it: eager, on another stream and captured, step after
    step against the definitions on what the cache then holds."""
    rng, heads, queries, depth, page, count, sequences = np.random.default_rng(8), 2, 8, 64, 8, 6, 3
    start, columns = np.array([150, 9, 79], np.int32), 24
    table, pages = pages_of(rng, [columns * page] * sequences, page)
    frequencies = device((10000.0 ** (-np.arange(32) / 32)).astype(np.float32))
    ctx, scale = context(), depth ** -0.5
    cache = cache_of(rng, pages, heads, page, depth, cache_tag)
    bounds = torch.zeros((pages, 2, heads, depth), dtype=torch.bfloat16, device=DEVICE)
    projected, positions = values(rng, (sequences, queries + 2 * heads, depth), tag), device(start)
    lengths, slots, pages_at = device(start + 1), torch.zeros(sequences, dtype=torch.int32, device=DEVICE), device(table)
    state = {}

    def bind(operation, inputs, outputs):
        bound = tio.Bound(ctx, operation, [tio.desc_of(t) for t in inputs])
        made = bound.outputs()
        made[:len(outputs)] = outputs
        return (lambda **how: bound.submit(inputs, made, **how)), made

    add, (_, rotated) = bind(hc.RotaryAppend(pages, page, tio.desc_of(cache).data_type, heads, HALF), [projected, positions, frequencies, slots], [cache])
    bound_all, _ = bind(hc.PageBounds(), [cache, pages_at, lengths], [bounds])
    bound_new, _ = bind(hc.PageBounds(1), [cache, pages_at, lengths], [bounds])
    select, (chosen, seen) = bind(hc.PagedSelect(count, page), [rotated, bounds, pages_at, lengths], [])
    attend, (out,) = bind(hc.PagedAttention(scale), [rotated, cache, chosen, seen], [])

    def step():
        for call in (add, bound_new, select, attend):
            call()

    lengths.copy_(device(start))
    note(f"steps of sparse decoding {tag} {cache_tag}")
    bound_all()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for turn in range(8):
        now = start + turn
        projected.copy_(values(rng, projected.shape, tag))
        positions.copy_(device(now))
        lengths.copy_(device(now + 1))
        slots.copy_(device(table[np.arange(sequences), now // page] * page + now % page))
        out.fill_(7.0)
        torch.cuda.synchronize()
        if turn < 2:
            step()
        elif turn == 2:
            with torch.cuda.stream(other):
                step()
        else:
            if "graph" not in state:
                state["graph"] = torch.cuda.CUDAGraph()
                with torch.cuda.graph(state["graph"], stream=other):
                    step()
                out.fill_(7.0)
                torch.cuda.synchronize()
            state["graph"].replay()
        torch.cuda.synchronize()
        with np.errstate(over="ignore"):
            held = cs.cache_values(cache)
        got_bounds = cs.bf16_bits(host(bounds).astype(np.float32))
        want_bounds = cs.page_bounds(held.astype(np.float32), table, now + 1, 0, got_bounds)
        assert (((got_bounds ^ want_bounds) == 0) | (((got_bounds | want_bounds) & 0x7FFF) == 0)).all()
        q = host(rotated)
        want_pages, want_seen = cs.selected(q[:, None], host(bounds), table, now + 1, heads, page, count)
        assert np.array_equal(chosen.cpu().numpy(), want_pages) and np.array_equal(seen.cpu().numpy(), want_seen)
        for i in range(sequences):
            for h in range(heads):
                place, mine = np.arange(want_seen[i, h]), slice(h * 4, h * 4 + 4)
                k, v = (held[want_pages[i, h, place // page], side, h, place % page][:, None] for side in (0, 1))
                want, _, bound, _ = attention_rows(q[i:i + 1, mine], k, v, int(want_seen[i, h]) - 1, True, 0, 0, scale, TYPES[tag])
                assert_within(out[i:i + 1, mine], want, bound)


@pytest.mark.parametrize("cache_tag,pages", [("mx4", 300_000), ("bf16", 70_000)])
def test_pages_beyond_32_bits(cache_tag, pages):
    """The last pages of a cache of more than 4 GiB, and the same in a small one."""
    rng, heads, queries, depth, page, tokens = np.random.default_rng(5), 8, 16, 128, 16, 200
    projected = values(rng, (tokens, queries + 2 * heads, depth), "bf16")
    positions, frequencies = torch.arange(tokens, dtype=torch.int32, device=DEVICE), device((10000.0 ** (-np.arange(64) / 64)).astype(np.float32))
    answers = []
    for count in (pages, 16):
        row = depth // 32 * 17 if cache_tag == "mx4" else depth
        cache = torch.zeros((count, 2, heads, page, row), dtype=TYPES[cache_tag], device=DEVICE)
        assert count == 16 or cache.numel() * cache.element_size() > 2 ** 32
        slots = torch.arange(count * page - tokens, count * page, dtype=torch.int32, device=DEVICE)
        table = torch.arange(count - 13, count, dtype=torch.int32, device=DEVICE)[None].contiguous()  # 200 tokens end a page: 8 places of the first are free
        note(f"pages beyond 32 bits {cache_tag} {count}")
        _, rotated = submit(hc.RotaryAppend(count, page, tio.desc_of(cache).data_type, heads, HALF), [projected, positions, frequencies, slots], [cache])
        lengths = torch.tensor([13 * page], dtype=torch.int32, device=DEVICE)
        (bounds,) = submit(hc.PageBounds(), [cache, table, lengths], [torch.zeros((count, 2, heads, depth), dtype=torch.bfloat16, device=DEVICE)])
        chosen, seen = submit(hc.PagedSelect(4, page), [rotated[-1:], bounds, table, lengths])
        (out,) = submit(hc.PagedAttention(0.1), [rotated[-1:], cache, chosen, seen])
        (whole,) = submit(hc.PagedAttention(0.1), [rotated[-1:], cache, table, lengths])
        answers.append((cache[-13:].clone(), bounds[-13:].clone(), chosen - count, seen, out, whole))
        del cache, bounds
        torch.cuda.empty_cache()
    for far, near in zip(*answers):
        assert torch.equal(far, near)
    assert (answers[0][4] != 0).any()


def test_an_output_within_an_operand_is_refused():
    cache = torch.zeros((4, 2, 2, 4, 64), dtype=torch.bfloat16, device=DEVICE)
    four, lengths = torch.zeros((2, 4), dtype=torch.int32, device=DEVICE), torch.zeros(2, dtype=torch.int32, device=DEVICE)
    rows, turns = cache[0].view(4, 4, 64), torch.zeros(32, dtype=torch.float32, device=DEVICE)
    bounds = cache.view(-1)[:4 * 2 * 2 * 64].view(4, 2, 2, 64)
    query = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device=DEVICE)
    for operation, inputs, outputs in ((hc.RotaryAppend(4, 4, hc.DataType.kBFloat16, 1), [rows[:2, :4], lengths, turns, lengths], [torch.zeros((4, 2, 1, 4, 64), dtype=torch.bfloat16, device=DEVICE), rows[:2, :2].contiguous()]),
                                       (hc.PageBounds(), [cache, four, lengths], [bounds]),
                                       (hc.PagedSelect(3, 4), [query, torch.zeros((4, 2, 2, 64), dtype=torch.bfloat16, device=DEVICE), four, lengths], [four.view(-1)[:8].view(2, 2, 2).new_zeros((2, 2, 3)), four.view(-1)[:4].view(2, 2)])):
        bound = tio.Bound(context(), operation, [tio.desc_of(t) for t in inputs])
        if isinstance(operation, hc.RotaryAppend):
            outputs[1] = rows.view(-1)[:2 * 2 * 64].view(2, 2, 64)
        note(f"outputs within operands of {type(operation).__name__}")
        with pytest.raises(hc.StatusError) as refused:
            bound.submit(inputs, outputs)
        assert refused.value.is_invalid_argument()
