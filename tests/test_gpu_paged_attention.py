"""PagedAppend and PagedAttention against the definition: every cache type, page size and order, ragged lengths, new tokens of
a few per sequence, windows with sinks, pages that are not there, free slots that hold no numbers; the two together with
Attention as a server runs them, eager, captured and on two streams."""
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

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
UNTOUCHED = 77.0


def values(rng, shape, dtype, std=1.0):
    x = torch.from_numpy(rng.normal(0, std, shape).astype(np.float32)).to(DEVICE)
    return x.to(torch.bfloat16).to(dtype) if dtype == torch.float8_e4m3fn else x.to(dtype)


def host(tensor):
    return tensor.double().cpu().numpy() if tensor.dtype != torch.float8_e4m3fn else tensor.float().double().cpu().numpy()


def words(tensor):
    return tensor.contiguous().view(torch.uint8)


# ---- PagedAppend ----------------------------------------------------------------------------
def append(keys, values_, slots, cache, **how):
    operation = hc.PagedAppend(cache.shape[0], cache.shape[3], tio.desc_of(cache).data_type)
    bound = tio.Bound(context(), operation, [tio.desc_of(t) for t in (keys, values_, slots)])
    bound.submit([keys, values_, slots], [cache], **how)
    torch.cuda.synchronize()


def narrowed(x, cache_type):
    return x.float().clamp(-448, 448).to(cache_type) if cache_type == torch.float8_e4m3fn else x


APPENDS = [(tag, cache, depth, page, tokens)
           for tag, cache in (("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "e4m3"), ("f16", "e4m3"), ("f32", "e4m3"))
           for depth, page, tokens in ((128, 16, 1), (64, 1, 37), (80, 24, 700), (63, 7, 41), (256, 64, 130), (72, 16, 33))]


@pytest.mark.parametrize("tag,cache_tag,depth,page,tokens", APPENDS)
def test_tokens_go_to_their_slots_and_nothing_else_changes(tag, cache_tag, depth, page, tokens):
    rng, heads, pages = np.random.default_rng(depth + tokens), 3, -(-tokens // page) + 2
    dtype, cache_type = TYPES[tag], TYPES[cache_tag]
    keys, vals = values(rng, (tokens, heads, depth), dtype, 3.0), values(rng, (tokens, heads, depth), dtype)
    cache = values(rng, (pages, 2, heads, page, depth), cache_type)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    for at, bad in zip(range(3, tokens, 9), (-1, pages * page, 2 ** 31 - 1, -2 ** 31)):
        slots[at] = bad
    want = words(cache).view(pages, 2, heads, page, -1).clone()
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < pages * page:
            want[slot // page, 0, :, slot % page] = words(narrowed(keys[t], cache_type)).view(heads, -1)
            want[slot // page, 1, :, slot % page] = words(narrowed(vals[t], cache_type)).view(heads, -1)
    note(f"append {tag} -> {cache_tag} depth {depth} page {page} tokens {tokens}")
    append(keys, vals, torch.from_numpy(slots).to(DEVICE), cache)
    assert torch.equal(words(cache).view(want.shape), want)


@pytest.mark.parametrize("tag", ["bf16", "f16"])
def test_every_pattern_to_e4m3(tag):
    """All 2^16 numbers of the type: nearest even, the largest for what is beyond it, NaN for NaN."""
    keys = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).to(DEVICE).view(TYPES[tag]).view(512, 1, 128)
    cache = torch.zeros((512, 2, 1, 1, 128), dtype=torch.uint8, device=DEVICE).view(torch.float8_e4m3fn)
    note(f"append of every pattern {tag}")
    append(keys, keys, torch.arange(512, dtype=torch.int32, device=DEVICE), cache)
    x = keys.float().view(-1)
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    for side in range(2):
        got = cache[:, side].float().view(-1)
        assert torch.equal(torch.isnan(got), torch.isnan(x))
        fine = ~torch.isnan(x)
        assert torch.equal(got[fine], want[fine])


def test_append_of_views_and_of_one_element_off():
    rng = np.random.default_rng(3)
    packed = values(rng, (50, 8, 64), torch.bfloat16)
    cache = torch.zeros((10, 2, 2, 8, 64), dtype=torch.bfloat16, device=DEVICE)
    slots = torch.randperm(80, device=DEVICE)[:50].to(torch.int32)
    note("append of views")
    for keys, vals in ((packed[:, 4:6], packed[:, 6:8]), (values(rng, (50 * 128 + 1,), torch.bfloat16)[1:].view(50, 2, 64),) * 2,
                       (packed[:1, 4:6].expand(50, -1, -1), packed.transpose(0, 1)[:2].transpose(0, 1))):
        append(keys, vals, slots, cache)
        where = slots.long()
        assert torch.equal(cache[where // 8, 0, :, where % 8], keys) and torch.equal(cache[where // 8, 1, :, where % 8], vals)


def test_two_tokens_of_one_slot_leave_one_of_them():
    rng = np.random.default_rng(4)
    keys, vals = values(rng, (40, 2, 128), torch.bfloat16), values(rng, (40, 2, 128), torch.bfloat16)
    cache = torch.zeros((4, 2, 2, 4, 128), dtype=torch.bfloat16, device=DEVICE)
    note("append twice into one slot")
    append(keys, vals, torch.full((40,), 5, dtype=torch.int32, device=DEVICE), cache)
    assert (cache[1, 0, 0, 1].expand(40, -1) == keys[:, 0]).all(1).any()
    cache[1, :, :, 1] = 0
    assert (cache == 0).all()


def test_append_into_its_own_operands_is_refused():
    cache = torch.zeros((4, 2, 2, 4, 128), dtype=torch.bfloat16, device=DEVICE)
    keys, slots = cache[0, 0], torch.zeros(2, dtype=torch.int32, device=DEVICE)
    bound = tio.Bound(context(), hc.PagedAppend(4, 4, hc.DataType.kBFloat16), [tio.desc_of(t) for t in (keys, keys, slots[:2])])
    note("append into its own operands")
    with pytest.raises(hc.StatusError) as refused:
        bound.submit([keys, keys, slots], [cache])
    assert refused.value.is_invalid_argument()


# ---- PagedAttention -------------------------------------------------------------------------
class Paged:
    """Sequences of keys and values in a cache whose pages are in no order; free slots hold `filler`."""

    def __init__(self, rng, lengths, heads, depth, page, cache_type, filler=0.5, spare=2, columns=None):
        held = [-(-max(0, n) // page) for n in lengths]
        self.pages, self.page = sum(held) + spare, page
        self.columns = max(held + [1]) if columns is None else columns
        order = rng.permutation(self.pages)
        self.cache = torch.full((self.pages, 2, heads, page, depth), filler, dtype=torch.bfloat16, device=DEVICE).to(cache_type)
        table = np.full((len(lengths), self.columns), -1, np.int32)
        self.keys, self.values, at = [], [], 0
        for i, n in enumerate(lengths):
            mine = order[at:at + held[i]]
            at += held[i]
            table[i, :held[i]] = mine[:self.columns]
            k, v = values(rng, (max(0, n), heads, depth), cache_type), values(rng, (max(0, n), heads, depth), cache_type)
            if n > 0:
                place = torch.arange(n, device=DEVICE)
                where = torch.from_numpy(mine.astype(np.int64)).to(DEVICE)[place // page]
                raw = words(self.cache).view(self.pages, 2, heads, page, -1)
                raw[where, 0, :, place % page] = words(k).view(n, heads, -1)
                raw[where, 1, :, place % page] = words(v).view(n, heads, -1)
            self.keys.append(k)
            self.values.append(v)
        self.table = torch.from_numpy(table).to(DEVICE)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)


def attend(operation, query, paged, cache=None):
    inputs = [query, paged.cache if cache is None else cache, paged.table, paged.lengths]
    bound = tio.Bound(context(), operation, [tio.desc_of(t) for t in inputs])
    outputs = [t.fill_(UNTOUCHED) for t in bound.outputs()]
    bound.submit(inputs, outputs)
    torch.cuda.synchronize()
    return outputs


def check(operation, query, paged, lengths, outputs, missing=()):
    """missing: per sequence, the keys whose page is not there."""
    rows = query if query.dim() == 4 else query[:, None]
    out = outputs[0].view(rows.shape)
    logs = outputs[1].view(rows.shape[:3]) if operation.return_log_sum else None
    for i, n in enumerate(lengths):
        n = max(0, n)
        known = min(n, paged.columns * paged.page)
        want, want_logs, bound, log_bound = attention_rows(host(rows[i]), host(paged.keys[i])[:known], host(paged.values[i])[:known], n - rows.shape[1], True,
                                                           operation.window, operation.sinks, operation.scale, query.dtype, missing[i] if missing else ())
        assert_within(out[i], want, bound)
        if logs is not None:
            assert_within(logs[i], want_logs, log_bound)


# type, cache, depth, query heads, key heads, page, lengths, new tokens, window, sinks, logarithms
DECODES = [
    ("bf16", "bf16", 128, 4, 1, 16, [1], 1, 0, 0, True),                                   # the first token
    ("bf16", "bf16", 128, 8, 2, 16, [1, 0, 17, 300, -3, 64], 1, 0, 0, True),               # some sequences hold nothing
    ("f16", "f16", 64, 2, 2, 1, [33, 5], 1, 0, 0, True),                                   # a page to a token
    ("bf16", "bf16", 256, 16, 2, 16, [700], 1, 0, 0, True),                                # few rows, a longer axis
    ("bf16", "bf16", 128, 8, 2, 16, [5000, 3], 1, 0, 0, True),
    ("f16", "f16", 80, 5, 1, 24, [100, 23, 24, 25], 4, 0, 0, True),                        # pages that end inside a tile
    ("bf16", "bf16", 128, 4, 2, 7, [200, 61], 3, 0, 0, False),
    ("bf16", "e4m3", 128, 8, 2, 64, [500, 63, 64, 65], 1, 0, 0, True),
    ("f16", "e4m3", 64, 4, 1, 16, [130, 7], 2, 0, 0, True),
    ("bf16", "e4m3", 256, 4, 2, 16, [333], 1, 0, 0, True),
    ("f16", "e4m3", 72, 2, 1, 24, [333, 100], 8, 0, 0, True),
    ("bf16", "bf16", 128, 16, 2, 16, [400, 90, 5], 8, 0, 0, True),                         # 64 rows to a key head
    ("f16", "f16", 96, 6, 3, 8, [300, 9], 16, 0, 0, False),                                # more new tokens than keys (9)
    ("bf16", "bf16", 128, 4, 1, 16, [1000, 30, 33], 1, 32, 0, True),                       # a window
    ("bf16", "bf16", 128, 4, 1, 16, [1000, 30, 37], 4, 32, 4, True),                       # and sinks
    ("f16", "f16", 64, 4, 2, 16, [900, 500], 2, 100, 70, True),                            # sinks past a tile
    ("bf16", "e4m3", 80, 4, 2, 24, [900, 500], 3, 333, 1, True),
    ("bf16", "bf16", 63, 2, 1, 16, [100], 2, 0, 0, True),                                  # no whole vectors
    ("f32", "f32", 64, 2, 1, 16, [100, 3], 2, 40, 1, True),
    ("f32", "e4m3", 64, 2, 1, 16, [100, 3], 1, 0, 0, True),
    ("bf16", "e4m3", 36, 2, 1, 16, [70], 1, 0, 0, False),
    ("bf16", "bf16", 64, 80, 1, 16, [200], 1, 0, 0, True),                                 # more heads to a key head than a tile
    ("bf16", "bf16", 128, 2, 1, 16, [260, 140], 100, 0, 0, True),                          # a chunk of a prompt
]


@pytest.mark.parametrize("case", DECODES, ids=[f"{c[0]}-{c[1]}-d{c[2]}-{c[3]}x{c[4]}-p{c[5]}-n{c[7]}-w{c[8]}s{c[9]}-{i}" for i, c in enumerate(DECODES)])
def test_new_tokens_over_a_paged_cache(case):
    tag, cache, depth, queries, heads, page, lengths, new, window, sinks, logs = case
    rng = np.random.default_rng(depth + 7 * new + len(lengths))
    paged = Paged(rng, lengths, heads, depth, page, TYPES[cache])
    query = values(rng, (len(lengths), new, queries, depth) if new != 1 else (len(lengths), queries, depth), TYPES[tag], 1.5)
    operation = hc.PagedAttention(depth ** -0.5, window, sinks, logs)
    note(f"paged attention {case}")
    check(operation, query, paged, lengths, attend(operation, query, paged))


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("depth", [64, 48, 128, 80, 256, 144])
@pytest.mark.parametrize("new,shared", [(1, 4), (3, 8), (8, 8)])
def test_rows_of_a_key_head_and_depths(cache, depth, new, shared):
    """16, 32 and 64 rows to a block, keys split and joined."""
    rng, lengths = np.random.default_rng(depth + new), [700, 33, 0]
    paged = Paged(rng, lengths, 2, depth, 16, TYPES[cache])
    query = values(rng, (3, new, 2 * shared, depth), torch.bfloat16, 1.5)
    note(f"paged attention {cache} depth {depth}, {new * shared} rows")
    for operation in (hc.PagedAttention(depth ** -0.5, return_log_sum=True), hc.PagedAttention(depth ** -0.5, 100, 3, True)):
        check(operation, query, paged, lengths, attend(operation, query, paged))
        rows = 16 if new * shared <= 16 else 32 if new * shared <= 32 else 64
        padded = 64 if depth <= 64 else 128 if depth <= 128 else 256
        label = f"attention_split/{'e4m3/' if cache == 'e4m3' else ''}{'d' if depth == padded else 'below-d'}{padded}/{rows}-rows"
        assert hc.last_launch_variant() == label + ("" if operation.window else f" + attention_join/d{padded}/row-to-block")


@pytest.mark.parametrize("depth", [64, 128, 256])
def test_many_rows_joined(depth):
    rng, lengths = np.random.default_rng(depth), [1, 900] + [20, 0, 140] * 13
    paged = Paged(rng, lengths, 4, depth, 16, torch.bfloat16)
    query = values(rng, (len(lengths), 4, 16, depth), torch.bfloat16, 1.5)
    operation = hc.PagedAttention(depth ** -0.5, return_log_sum=True)
    note(f"paged attention of {len(lengths)} sequences of 64 rows, depth {depth}")
    check(operation, query, paged, lengths, attend(operation, query, paged))
    assert hc.last_launch_variant().endswith(f"attention_join/d{depth}/rows")


@pytest.mark.parametrize("window,sinks", [(1, 0), (31, 0), (33, 1), (128, 130), (200, 31), (5000, 7)])
def test_windows_at_every_offset(window, sinks):
    """Windows that begin anywhere in a step, over sinks that end anywhere before them."""
    rng, lengths = np.random.default_rng(window), list(range(1, 24, 3)) + list(range(150, 400, 23))
    paged = Paged(rng, lengths, 1, 64, 16, torch.bfloat16)
    query = values(rng, (len(lengths), 2, 2, 64), torch.bfloat16, 1.5)
    operation = hc.PagedAttention(0.125, window, sinks, True)
    note(f"paged attention windows {window} {sinks}")
    check(operation, query, paged, lengths, attend(operation, query, paged))


def test_many_sequences_of_every_length():
    rng = np.random.default_rng(21)
    lengths = [int(n) for n in rng.integers(0, 400, 150)] + [3000]
    paged = Paged(rng, lengths, 1, 64, 16, torch.bfloat16)
    query = values(rng, (len(lengths), 2, 64), torch.bfloat16, 1.5)
    operation = hc.PagedAttention(0.125, return_log_sum=True)
    note("paged attention of 151 sequences")
    check(operation, query, paged, lengths, attend(operation, query, paged))


@pytest.mark.parametrize("tag,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3")])
@pytest.mark.parametrize("depth,new", [(128, 1), (256, 1), (80, 3), (64, 20)])
def test_free_slots_that_hold_no_numbers(tag, cache, depth, new):
    rng, lengths = np.random.default_rng(22), [70, 33, 1]
    paged = Paged(rng, lengths, 2, depth, 16, TYPES[cache], filler=math.nan)
    query = values(rng, (3, new, 4, depth), TYPES[tag], 1.5)
    operation = hc.PagedAttention(depth ** -0.5, return_log_sum=True)
    note(f"paged attention with NaN in free slots {tag} {cache} {depth} {new}")
    check(operation, query, paged, lengths, attend(operation, query, paged))


@pytest.mark.parametrize("tag", ["bf16", "f16"])
@pytest.mark.parametrize("depth", [64, 128, 256])
@pytest.mark.parametrize("queries", [2, 8, 16])
def test_new_tokens_do_not_see_those_behind_them(tag, depth, queries):
    """The last new token's key and value are no numbers, and one key before the window of all but the first."""
    rng, lengths = np.random.default_rng(23), [100]
    paged = Paged(rng, lengths, 1, depth, 16, TYPES[tag])
    place = (int(paged.table[0, 99 // 16]), 99 % 16), (int(paged.table[0, 64 // 16]), 64 % 16)
    for page, at in place:
        paged.cache[page, 0, 0, at], paged.cache[page, 1, 0, at] = math.nan, math.inf
    query = values(rng, (1, 4, queries, depth), TYPES[tag], 1.5)
    operation = hc.PagedAttention(depth ** -0.5, 32)
    note(f"paged attention of new tokens with NaN behind them {tag} {depth} {queries}")
    (out,) = attend(operation, query, paged)
    keys, vals = host(paged.keys[0]), host(paged.values[0])
    want, _, bound, _ = attention_rows(host(query[0]), keys, vals, 96, True, 32, 0, operation.scale, query.dtype)
    assert_within(out[0, :3], want[:3], bound[:3])  # queries 96..98 see keys from 65 on
    assert torch.isnan(out[0, 3]).all()


@pytest.mark.parametrize("tag", ["bf16", "f16"])
@pytest.mark.parametrize("queries", [2, 8, 16])
def test_an_infinite_value_reaches_the_rows_that_see_it(tag, queries):
    """Alone in a sequence's first key, among others, and in the newest of four tokens."""
    rng, lengths = np.random.default_rng(28), [4, 60]
    paged = Paged(rng, lengths, 1, 64, 16, TYPES[tag])
    paged.cache[int(paged.table[0, 0]), 1, 0, 0, 5] = math.inf
    paged.cache[int(paged.table[1, 3]), 1, 0, 58 % 16, 6] = -math.inf
    query = values(rng, (2, 4, queries, 64), TYPES[tag])
    note(f"paged attention of infinite values {tag} {queries}")
    (out,) = attend(hc.PagedAttention(0.125), query, paged)
    assert (out[0, :, :, 5] == math.inf).all() and (out[1, 2:, :, 6] == -math.inf).all()
    out[0, :, :, 5], out[1, 2:, :, 6] = 0, 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("tag,cache", [("bf16", "bf16"), ("f16", "e4m3"), ("f32", "f32")])
def test_pages_that_are_not_there_hold_no_keys(tag, cache):
    rng, lengths = np.random.default_rng(24), [100, 40, 64, 500]
    paged = Paged(rng, lengths, 2, 64, 16, TYPES[cache])
    missing = [[], [], [], []]
    for i, column, page in ((0, 2, -1), (0, 6, 2 ** 31 - 1), (1, 0, -2 ** 31), (1, 1, paged.pages), (1, 2, -7), (3, 5, paged.pages + 1)):
        paged.table[i, column] = page
        missing[i] += list(range(column * 16, (column + 1) * 16))
    query = values(rng, (4, 4, 64), TYPES[tag], 1.5)
    operation = hc.PagedAttention(0.125, return_log_sum=True)
    note(f"paged attention with pages that are not there {tag} {cache}")
    check(operation, query, paged, lengths, attend(operation, query, paged), missing)


def test_lengths_past_the_table_and_a_table_of_views():
    """Keys past the last column do not exist; positions still count from the length.  The table's rows lie apart."""
    rng, lengths = np.random.default_rng(25), [100, 20]
    paged = Paged(rng, lengths, 2, 64, 16, torch.bfloat16, columns=3)
    wide = torch.full((2, 11), -1, dtype=torch.int32, device=DEVICE)
    wide[:, 4:7] = paged.table
    paged.table = wide[:, 4:7]
    query = values(rng, (2, 4, 64), torch.bfloat16)
    note("paged attention of lengths past the table")
    for operation in (hc.PagedAttention(0.125, return_log_sum=True), hc.PagedAttention(0.125, 60, 2, return_log_sum=True)):
        check(operation, query, paged, lengths, attend(operation, query, paged))
    paged.lengths[0] = 2 ** 31 - 1
    operation = hc.PagedAttention(0.125, return_log_sum=True)
    check(operation, query, paged, [2 ** 31 - 1, 20], attend(operation, query, paged))


@pytest.mark.parametrize("tag,cache", [("bf16", "bf16"), ("bf16", "e4m3")])
def test_caches_of_other_layouts(tag, cache):
    """The tokens in front of the heads, keys and values apart, one page to a sequence: strides of the cache's descriptor."""
    rng, lengths = np.random.default_rng(26), [90, 31]
    paged = Paged(rng, lengths, 2, 64, 16, TYPES[cache])
    query = values(rng, (2, 4, 64), TYPES[tag], 1.5)
    operation = hc.PagedAttention(0.125, return_log_sum=True)
    note(f"paged attention over other layouts {cache}")
    raw = words(paged.cache).view(paged.cache.shape[:4] + (-1,))
    for order in ((0, 1, 3, 2, 4), (1, 0, 2, 3, 4), (1, 3, 0, 2, 4)):
        back = [order.index(a) for a in range(5)]
        other = raw.permute(order).contiguous().view(TYPES[cache]).permute(back)
        assert other.stride() != paged.cache.stride()
        check(operation, query, paged, lengths, attend(operation, query, paged, other))
    whole = torch.zeros((2, 2, 2, 90, 64), dtype=torch.uint8, device=DEVICE) if cache == "e4m3" else torch.zeros((2, 2, 2, 90, 64), dtype=TYPES[cache], device=DEVICE)
    for i, n in enumerate(lengths):
        for side, held in enumerate((paged.keys[i], paged.values[i])):
            whole[i, side, :, :n] = (words(held).view(held.shape) if cache == "e4m3" else held).transpose(0, 1)
    contiguous = Paged(rng, [1], 2, 64, 16, TYPES[cache])
    contiguous.cache, contiguous.page, contiguous.columns = whole.view(TYPES[cache]), 90, 1
    contiguous.keys, contiguous.values, contiguous.lengths = paged.keys, paged.values, paged.lengths
    contiguous.table = torch.arange(2, dtype=torch.int32, device=DEVICE)[:, None]
    check(operation, query, contiguous, lengths, attend(operation, query, contiguous))


def test_caches_of_more_than_32_bits_of_bytes():
    rng = np.random.default_rng(27)
    if torch.cuda.mem_get_info()[0] < 16 * 2 ** 30:
        pytest.skip("needs memory for a cache of some GiB")
    note("append and paged attention past 4 GiB and 2^31 elements")
    cache = torch.zeros((2 ** 17 + 40, 2, 1, 64, 256), dtype=torch.bfloat16, device=DEVICE)
    order = [2 ** 17 + 39, 5, 2 ** 17 + 2, 2 ** 16 + 1]
    keys, vals = values(rng, (200, 1, 256), torch.bfloat16), values(rng, (200, 1, 256), torch.bfloat16)
    slots = torch.tensor([order[t // 64] * 64 + t % 64 for t in range(200)], dtype=torch.int32, device=DEVICE)
    append(keys, vals, slots, cache)
    paged = Paged(rng, [1], 1, 256, 64, torch.bfloat16)
    paged.cache, paged.columns, paged.keys, paged.values = cache, 4, [keys], [vals]
    paged.table = torch.tensor([order], dtype=torch.int32, device=DEVICE)
    paged.lengths = torch.tensor([200], dtype=torch.int32, device=DEVICE)
    query = values(rng, (1, 2, 256), torch.bfloat16, 1.5)
    operation = hc.PagedAttention(0.0625)
    check(operation, query, paged, [200], attend(operation, query, paged))


# ---- together -------------------------------------------------------------------------------
class Layer:
    """One layer's attention as a server runs it: prompts packed into Attention and appended, then a step at a time."""

    def __init__(self, rng, cache_tag, window=0, sinks=0):
        self.prompts, self.steps, self.heads, self.queries, self.depth, self.page = [45, 1, 130], 5, 2, 8, 128, 16
        self.window, self.sinks = window, sinks
        total = sum(self.prompts)
        dtype = torch.bfloat16
        make = lambda *shape: values(rng, shape, dtype, 1.2)  # noqa: E731
        self.query, self.key, self.value = make(total, self.queries, self.depth), make(total, self.heads, self.depth), make(total, self.heads, self.depth)
        n = len(self.prompts)
        self.step_query = make(self.steps, n, self.queries, self.depth)
        self.step_key, self.step_value = make(self.steps, n, self.heads, self.depth), make(self.steps, n, self.heads, self.depth)
        columns = -(-(max(self.prompts) + self.steps) // self.page)
        self.cache = torch.full((n * columns + 1, 2, self.heads, self.page, self.depth), math.nan, dtype=dtype, device=DEVICE).to(TYPES[cache_tag])
        table = rng.permutation(n * columns + 1)[:n * columns].reshape(n, columns).astype(np.int32)
        self.table = torch.from_numpy(table).to(DEVICE)
        self.offsets = torch.tensor(np.concatenate([[0], np.cumsum(self.prompts)]), dtype=torch.int32, device=DEVICE)
        slot = lambda i, place: int(table[i, place // self.page]) * self.page + place % self.page  # noqa: E731
        self.slots = torch.tensor([slot(i, p) for i, length in enumerate(self.prompts) for p in range(length)], dtype=torch.int32, device=DEVICE)
        self.step_slots = torch.tensor([[slot(i, length + s) for i, length in enumerate(self.prompts)] for s in range(self.steps)], dtype=torch.int32, device=DEVICE)
        self.step_lengths = torch.tensor([[length + s + 1 for length in self.prompts] for s in range(self.steps)], dtype=torch.int32, device=DEVICE)
        scale, kind = self.depth ** -0.5, tio.desc_of(self.cache).data_type
        bind = lambda operation, *inputs: tio.Bound(context(), operation, [tio.desc_of(t) for t in inputs])  # noqa: E731
        self.attention = bind(hc.Attention(scale, True, window, sinks), self.query, self.key, self.value, self.offsets)
        self.fill = bind(hc.PagedAppend(self.cache.shape[0], self.page, kind), self.key, self.value, self.slots)
        self.append = bind(hc.PagedAppend(self.cache.shape[0], self.page, kind), self.step_key[0], self.step_value[0], self.step_slots[0])
        self.decode = bind(hc.PagedAttention(scale, window, sinks), self.step_query[0], self.cache, self.table, self.step_lengths[0])
        self.out = self.attention.outputs()[0]
        self.step_out = torch.zeros_like(self.step_query)

    def submit(self):
        self.attention.submit([self.query, self.key, self.value, self.offsets], [self.out])
        self.fill.submit([self.key, self.value, self.slots], [self.cache])
        for s in range(self.steps):
            self.append.submit([self.step_key[s], self.step_value[s], self.step_slots[s]], [self.cache])
            self.decode.submit([self.step_query[s], self.cache, self.table, self.step_lengths[s]], [self.step_out[s]])

    def check(self):
        cast = lambda t: host(narrowed(t, self.cache.dtype))  # noqa: E731
        first = 0
        for i, length in enumerate(self.prompts):
            span = slice(first, first + length)
            first += length
            scale = self.depth ** -0.5
            want, _, bound, _ = attention_rows(host(self.query[span]), host(self.key[span]), host(self.value[span]), 0, True, self.window, self.sinks, scale, torch.bfloat16)
            assert_within(self.out[span], want, bound)
            keys = np.concatenate([cast(self.key[span]), cast(self.step_key[:, i])])
            vals = np.concatenate([cast(self.value[span]), cast(self.step_value[:, i])])
            want, _, bound, _ = attention_rows(host(self.step_query[:, i]), keys, vals, length, True, self.window, self.sinks, scale, torch.bfloat16)
            assert_within(self.step_out[:, i], want, bound)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_prompts_then_steps(cache, window, sinks):
    layer = Layer(np.random.default_rng(31), cache, window, sinks)
    note(f"a layer's prompts and steps {cache} {window} {sinks}")
    layer.submit()
    torch.cuda.synchronize()
    layer.check()


def test_a_captured_layer_replays_bit_identically():
    layer = Layer(np.random.default_rng(32), "bf16")
    note("a layer eager, then captured")
    layer.submit()
    torch.cuda.synchronize()
    want = [t.clone() for t in (layer.out, layer.step_out, layer.cache)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.submit()
    for replay in range(3):
        note(f"replay {replay} of a layer")
        layer.out.zero_(), layer.step_out.zero_(), layer.cache.fill_(math.nan)
        for bound in (layer.attention, layer.fill, layer.append, layer.decode):
            if bound.workspace is not None:
                bound.workspace.fill_(0xFF if replay % 2 else 0)
        assert np.isfinite(torch.randn(1 << 20, device=DEVICE).sum().item())
        graph.replay()
        torch.cuda.synchronize()
        for t, expected in zip((layer.out, layer.step_out, layer.cache), want):
            assert torch.equal(words(t), words(expected))


def test_two_layers_at_once_on_two_streams():
    layers = [Layer(np.random.default_rng(33 + i), "bf16") for i in range(2)]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    note("two layers on two streams")
    for layer, stream in zip(layers, streams):
        with torch.cuda.stream(stream):
            layer.submit()
    torch.cuda.synchronize()
    for layer in layers:
        layer.check()


def test_static_scratch_serves_the_same_bits():
    rng, lengths = np.random.default_rng(35), [700, 20, 3000]
    paged = Paged(rng, lengths, 2, 128, 16, torch.bfloat16)
    query = values(rng, (3, 8, 128), torch.bfloat16)
    inputs = [query, paged.cache, paged.table, paged.lengths]
    bound = tio.Bound(context(), hc.PagedAttention(0.088), [tio.desc_of(t) for t in inputs])
    assert bound.prepared.workspace_requirement().size <= hc.capi.load().hyle_hip_static_scratch_bytes()
    note("paged attention through the library's scratch")
    (want,), (got,) = bound.outputs(), bound.outputs()
    bound.submit(inputs, [want])
    bound.prepared.create_invocation_without_workspace().submit_without_workspace(tio.current_stream_handle(), [t.data_ptr() for t in inputs], [got.data_ptr()])
    torch.cuda.synchronize()
    assert torch.equal(want, got)
