"""The cache's operators where one of their forms alone can go wrong: scores that are no numbers in every kernel that takes them, several tiles of pages
to a wave, keys in 4 bits that are no numbers, seen and hidden, and more new tokens than a tile of rows holds."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyle_amd import compute as hc

import cache_support as cs
from attention_support import assert_within, attention_rows
from gpu_support import DEVICE, note
from test_gpu_cache_operators import TYPES, bounds_of, cache_of, device, host, off_by, pages_of, submit, values

pytestmark = pytest.mark.gpu


def i32(numbers):
    return torch.tensor(numbers, dtype=torch.int32, device=DEVICE)


# ---- scores ----------------------------------------------------------------------------------
def assert_chosen(query, bounds, table, lengths, heads, page, counts):
    for count in counts:
        got = submit(hc.PagedSelect(count, page), [query, bounds, device(table), i32(lengths)])
        with np.errstate(all="ignore"):
            want = cs.selected(host(query), host(bounds), table, lengths, heads, page, count)
        assert np.array_equal(got[0].cpu().numpy(), want[0]), count
        assert np.array_equal(got[1].cpu().numpy(), want[1]), count


def plant(bounds, query, table, heads, shared, depth):
    """Bounds that are no finite numbers, in either half of the depth, of the first and of a later key head: sums that are infinite of both signs,
    that are no numbers, and that are finite beside one that is not."""
    inf, nan = float("inf"), float("nan")
    ends, last = (0, 5, depth // 2 - 1, depth // 2, depth - 1), heads - 1
    for i, d in enumerate(ends):
        at = table[0, 3 + 4 * i:7 + 4 * i].astype(np.int64)
        bounds[int(at[0]), 1, 0, d] = nan
        bounds[int(at[1]), 1, last, d] = inf
        bounds[int(at[2]), 0, last, d] = -inf
        bounds[int(at[3]), 0, 0, d] = -inf
    whole = table[0, 30:34].astype(np.int64)
    bounds[int(whole[0]), 1] = inf
    bounds[int(whole[1]), 0] = -inf                                                        # inf - inf with queries of both signs
    bounds[int(whole[2]), 0], bounds[int(whole[2]), 1] = inf, -inf                          # a page whose keys are no numbers
    bounds[int(whole[3]), 0, 0, 1], bounds[int(whole[3]), 1, 0, depth - 2] = -inf, inf
    if query.shape[0] > 1:
        row = min(query.shape[1] * shared - 1, 4 + (16 if query.shape[1] * shared > 16 else 0))  # of a second step of rows, where there is one
        query[1, row // shared, last * shared + row % shared, depth // 2 + 1] = nan
    if query.shape[0] > 2:
        query[2, 0, 0, 0], query[2, -1, shared - 1, depth - 1] = inf, -inf
        query[2, :, last * shared:] *= (torch.arange(depth, device=DEVICE) % 2)            # zeros, which infinite bounds make no numbers of


@pytest.mark.parametrize("tag", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("depth,off", [(64, 0), (96, 0), (128, 0), (136, 0), (256, 0), (128, 2), (33, 0)])
@pytest.mark.parametrize("shared,new", [(2, 1), (7, 1), (6, 2), (17, 2)])
def test_scores_that_are_no_numbers(tag, depth, off, shared, new):
    """Of up to 4, 8, 16 and more query rows to a key head, by halves of the depth where it is over 128, padded, and without vectors."""
    rng, heads, page, lengths = np.random.default_rng(depth + 10 * shared), 2, 8, (900, 700, 811, 40, 1)
    table, pages = pages_of(rng, lengths, page)
    bounds, query = bounds_of(rng, pages, heads, depth), values(rng, (5, new, heads * shared, depth), tag)
    plant(bounds, query, table, heads, shared, depth)
    table[1, 4:60:7], table[1, 5:60:11] = -1, pages
    bounds = off_by(bounds, off) if off else bounds
    note(f"scores that are no numbers {tag} depth {depth} off {off} rows {shared} x {new}")
    assert_chosen(query, bounds, table, lengths, heads, page, (4, 17, 24, 40, 112))


@pytest.mark.parametrize("tag,depth,shared,new", [("bf16", 256, 2, 1), ("f16", 256, 6, 2), ("bf16", 128, 4, 1), ("f32", 136, 5, 1), ("bf16", 96, 3, 4),
                                                  ("f16", 64, 2, 2), ("bf16", 64, 9, 1)])
def test_several_tiles_of_pages_to_a_wave(tag, depth, shared, new):
    """Pages of one key each, of so many key heads that a wave takes tile after tile, sequences that end in each of them."""
    rng, heads, sequences = np.random.default_rng(depth + shared), 8, 24
    lengths = tuple(int(n) for n in np.concatenate(([1500, 1, 0, 65], rng.integers(60, 1500, sequences - 4))))
    table, pages = pages_of(rng, lengths, 1)
    bounds, query = bounds_of(rng, pages, heads, depth), values(rng, (sequences, new, heads * shared, depth), tag)
    plant(bounds, query, table, heads, shared, depth)
    table[5, 9:50:4] = -1
    note(f"several tiles of pages to a wave {tag} depth {depth} rows {shared} x {new}")
    assert_chosen(query, bounds, table, lengths, heads, 1, (12, 140))


# ---- keys in 4 bits that are no numbers -------------------------------------------------------
KEYS_4 = [("bf16", 128, 8, 2, 1), ("f16", 96, 8, 2, 3), ("bf16", 256, 8, 1, 2), ("f16", 64, 24, 1, 1), ("bf16", 32, 6, 2, 3), ("bf16", 128, 32, 1, 2),
          ("f16", 224, 20, 1, 3), ("f32", 64, 6, 3, 3)]


@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3)])
@pytest.mark.parametrize("tag,depth,queries,heads,new", KEYS_4)
def test_keys_in_four_bits_that_are_no_numbers(tag, depth, queries, heads, new, window, sinks):
    """A key whose scale is 255 makes the rows that see it no numbers.  Others are as they are without: of the last new token, before a window, behind
    the sequence's end in its last page, and in the page that stands for those that are not there."""
    rng, page, lengths = np.random.default_rng(depth + queries), 16, (300, 131, 700, 40, 290, 0, 1, 17)
    table, pages = pages_of(rng, lengths, page, spare=3)
    spare = next(i for i in range(pages) if i not in table)  # page 0 is in no table
    table = np.where(table == 0, spare, table)
    cache = cache_of(rng, pages, heads, page, depth, "mx4")
    raw = cache.cpu().numpy()
    scales = cs.mx4_split(raw)[1]
    scales[0] = 255
    for i, n in enumerate(lengths):
        if n % page:
            scales[table[i, n // page], :, :, n % page:] = 255
    gone = {1: (2, 5), 4: (0, 17)}
    for i, columns in gone.items():
        table[i, list(columns)] = (-1, pages)

    def mark(i, key, block):
        scales[table[i, key // page], 0, :, key % page, block] = 255

    blocks = depth // 32
    mark(0, lengths[0] - 1, blocks - 1)          # seen by the last token alone
    mark(2, 5, 0)                                # seen by all, or before the window
    mark(3, 20, blocks // 2)                     # in the middle of one that a window holds
    mark(4, 289, 0), mark(4, 100, blocks - 1)
    mark(6, 0, 0)                                # the only one
    for key in range(17):                        # all of them
        mark(7, key, key % blocks)
    query, cache = values(rng, (len(lengths), new, queries, depth), tag, 0.7), device(raw)
    note(f"keys in 4 bits that are no numbers {tag} depth {depth} heads {queries}/{heads} new {new} window {window}")
    outputs = submit(hc.PagedAttention(0.1, window, sinks, True), [query, cache, device(table), i32(lengths)])
    held = cs.cache_values(cache)
    for i, n in enumerate(lengths):
        place = np.arange(n)
        at = np.clip(table[i, place // page], 0, pages - 1)
        k, v = (held[at, side, :, place % page] for side in (0, 1))
        missing = np.flatnonzero((table[i, place // page] < 0) | (table[i, place // page] >= pages))
        k[missing], v[missing] = 0.0, 0.0
        with np.errstate(invalid="ignore"):
            want, logs, bound, log_bound = attention_rows(host(query[i]), k, v, n - new, True, window, sinks, 0.1, query.dtype, missing)
        assert_within(outputs[0][i], want, bound)
        assert_within(outputs[1][i], logs, log_bound)
        assert np.isnan(want[-1]).all() == (i in (0, 3, 4, 6, 7) or (i == 2 and window == 0))


# ---- many new tokens, tables without columns, the same twice -----------------------------------
@pytest.mark.parametrize("tag,cache_tag,depth,queries,heads,new,window,sinks", [
    ("bf16", "mx4", 128, 16, 2, 40, 0, 0), ("f16", "mx4", 64, 6, 2, 30, 100, 4), ("bf16", "mx4", 96, 12, 1, 17, 64, 0), ("f16", "mx4", 256, 10, 2, 33, 0, 0)])
@pytest.mark.parametrize("apart", [False, True])
def test_more_new_tokens_than_a_tile_of_rows(tag, cache_tag, depth, queries, heads, new, window, sinks, apart):
    """Chunks of prompts over a cache in 4 bits, of pages of the sequence and of each key head."""
    rng, page, lengths, shared = np.random.default_rng(depth + new), 16, (700, new, 333, 5), queries // heads
    table, pages = pages_of(rng, lengths, page)
    cache = cache_of(rng, pages, heads, page, depth, cache_tag)
    query = values(rng, (len(lengths), new, queries, depth), tag, 0.7)
    tables = np.repeat(table[:, None], heads, axis=1)
    seen = np.repeat(np.array(lengths, np.int32)[:, None], heads, axis=1)
    if apart:
        tables[0, -1, :20] = tables[0, -1, 20:40]                 # a head with other pages, and fewer
        seen[0, -1], seen[2, 0] = 401, 333 - 2 * page
    note(f"many new tokens {tag} {cache_tag} depth {depth} heads {queries}/{heads} new {new} window {window} apart {apart}")
    outputs = submit(hc.PagedAttention(0.1, window, sinks, True),
                     [query, cache, device(tables if apart else table), device(seen) if apart else i32(lengths)])
    held = cs.cache_values(cache)
    for i in range(len(lengths)):
        for h in range(heads):
            n, mine = int(seen[i, h]), slice(h * shared, (h + 1) * shared)
            place = np.arange(n)
            k, v = (held[tables[i, h, place // page], side, h, place % page][:, None] for side in (0, 1))
            want, logs, bound, log_bound = attention_rows(host(query[i])[:, mine], k, v, n - new, True, window, sinks, 0.1, query.dtype)
            assert_within(outputs[0][i, :, mine], want, bound)
            assert_within(outputs[1][i, :, mine], logs, log_bound)


@pytest.mark.parametrize("cache_tag", ["bf16", "mx4"])
def test_no_columns_for_any_key_head(cache_tag):
    rng = np.random.default_rng(4)
    cache, query = cache_of(rng, 3, 2, 16, 64, cache_tag), values(rng, (3, 2, 4, 64), "bf16")
    note(f"no columns for any key head {cache_tag}")
    out, logs = submit(hc.PagedAttention(0.1, return_log_sum=True), [query, cache, torch.zeros((3, 2, 0), dtype=torch.int32, device=DEVICE), i32([[5, 0], [1, -1], [700, 2]])])
    assert (out == 0).all() and torch.isneginf(logs).all()


@pytest.mark.parametrize("tag,cache_tag,depth", [("bf16", "mx4", 128), ("f16", "mx4", 256), ("bf16", "bf16", 128), ("bf16", "e4m3", 64)])
def test_the_same_call_gives_the_same_bits(tag, cache_tag, depth):
    """Chunks are joined in their order, whatever block ends first."""
    rng, heads, lengths = np.random.default_rng(depth), 2, (9000, 40, 3001)
    table, pages = pages_of(rng, lengths, 16)
    cache, query = cache_of(rng, pages, heads, 16, depth, cache_tag), values(rng, (3, 2, 8, depth), tag)
    bounds = bounds_of(rng, pages, heads, depth)
    seen = []
    for turn in range(4):
        note(f"the same call {cache_tag} depth {depth} turn {turn}")
        whole = submit(hc.PagedAttention(0.1, return_log_sum=True), [query, cache, device(table), i32(lengths)])
        chosen = submit(hc.PagedSelect(60, 16), [query, bounds, device(table), i32(lengths)])
        part = submit(hc.PagedAttention(0.1, return_log_sum=True), [query, cache, *chosen])
        seen.append([*whole, *chosen, *part])
    for others in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], others))
