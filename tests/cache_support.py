"""The cache's operators in numpy for the tests: 4-bit blocks, the rotation, a page's bounds, the choice of pages."""
from __future__ import annotations

import numpy as np
import torch

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mx4_encode(x: np.ndarray, dtype=torch.bfloat16):
    """Rows [.., depth] in float64 as codes [.., depth / 2] and scales [.., depth / 32]: the definition, level by level."""
    blocks = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(blocks).all(-1)
    blocks = np.where(bad[..., None], 0.0, blocks)
    fraction, exponent = np.frexp(np.abs(blocks).max(-1))  # fraction in [0.5, 1)
    power = np.where(fraction == 0, -127, exponent - 1 - 2 + (2 * fraction > 1.75))
    power = np.clip(power, -127, 13 if dtype == torch.float16 else 125)
    y = blocks / np.ldexp(1.0, power)[..., None]
    away = np.abs(np.abs(y)[..., None] - LEVELS)
    # of two levels at the same distance the even one comes first
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])
    code = order[np.argmin(away[..., order], axis=-1)].astype(np.uint8) | (np.signbit(y).astype(np.uint8) << 3)
    code = np.where(bad[..., None], 0, code).reshape(*x.shape[:-1], -1).astype(np.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, np.where(bad, 255, power + 127).astype(np.uint8)


def mx4_decode(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    code = np.stack((codes & 15, codes >> 4), axis=-1).reshape(*codes.shape[:-1], -1)
    value = np.where(code >= 8, -1.0, 1.0) * LEVELS[code & 7]
    factor = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return value * np.repeat(factor, 32, axis=-1)


def mx4_join(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """[.., page, depth / 2] and [.., page, depth / 32] as a cache's bytes [.., page, 17 depth / 32]."""
    lead, page = codes.shape[:-2], codes.shape[-2]
    flat = np.concatenate((codes.reshape(*lead, -1), scales.reshape(*lead, -1)), axis=-1)
    return flat.reshape(*lead, page, codes.shape[-1] + scales.shape[-1])


def mx4_split(cache: np.ndarray):
    """A cache's bytes as codes and scales, views."""
    lead, page, row = cache.shape[:-2], cache.shape[-2], cache.shape[-1]
    depth = row // 17 * 32
    flat = cache.reshape(*lead, page * row)
    return flat[..., :page * depth // 2].reshape(*lead, page, depth // 2), flat[..., page * depth // 2:].reshape(*lead, page, depth // 32)


def cache_values(cache: torch.Tensor) -> np.ndarray:
    """[pages, 2, heads, page, depth] in float64, whatever the cache keeps."""
    if cache.dtype == torch.uint8:
        return mx4_decode(*mx4_split(np.ascontiguousarray(cache.cpu().numpy())))
    return cache.cpu().double().numpy()


def rotated(x: np.ndarray, positions, frequencies: np.ndarray, half_split: bool) -> np.ndarray:
    """Rows [tokens, heads, depth] in float32, every product and sum rounded; cos and sin of the f32 phase from 64 bits."""
    x = np.asarray(x, np.float32)
    out = x.copy()
    pairs = frequencies.shape[-1]
    phase = (np.asarray(frequencies, np.float32) * np.asarray(positions).astype(np.float32)[:, None]).astype(np.float32)
    c = np.cos(phase.astype(np.float64)).astype(np.float32)[:, None]
    s = np.sin(phase.astype(np.float64)).astype(np.float32)[:, None]
    first = slice(0, pairs) if half_split else slice(0, 2 * pairs, 2)
    second = slice(pairs, 2 * pairs) if half_split else slice(1, 2 * pairs, 2)
    a, b = x[..., first], x[..., second]
    out[..., first] = a * c - b * s
    out[..., second] = a * s + b * c
    return out


def bf16_bits(x: np.ndarray) -> np.ndarray:
    return (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def page_bounds(values: np.ndarray, table: np.ndarray, lengths, newest: int, before: np.ndarray) -> np.ndarray:
    """Bounds [pages, 2, heads, depth] as bf16 bits: `before` where no page is written."""
    out = before.copy()
    pages, _, _, page, _ = values.shape
    for row, length in zip(table, lengths):
        first = 0 if newest == 0 else max(0, length - newest) // page
        for column in range(first, min(len(row), -(-max(length, 0) // page))):
            if not 0 <= row[column] < pages:
                continue
            keys = values[row[column], 0, :, :min(page, length - column * page)]
            low = np.where(np.isnan(keys), np.inf, keys).min(1)
            high = np.where(np.isnan(keys), -np.inf, keys).max(1)
            out[row[column], 0] = _outward(low, -np.inf)
            out[row[column], 1] = _outward(high, np.inf)
    return out


def _outward(x: np.ndarray, towards: float) -> np.ndarray:
    """The nearest bf16 number that is x or lies on that side of it."""
    bits = bf16_bits(x.astype(np.float32))  # towards zero
    value = (bits.astype(np.uint32) << 16).view(np.float32)
    short = (value > x) if towards < 0 else (value < x)
    return np.where(short, bits + 1, bits).astype(np.uint16)  # away from zero, where x is


def selected(query: np.ndarray, bounds: np.ndarray, table: np.ndarray, lengths, heads: int, page: int, count: int):
    """Chosen pages [B, H, count] and lengths [B, H]: query [B, R, Hq, D], bounds [pages, 2, H, D], both in float64."""
    sequences, rows, queries, _ = query.shape
    shared, columns = queries // heads, table.shape[1]
    out = np.full((sequences, heads, count), -1, np.int32)
    seen = np.zeros((sequences, heads), np.int32)
    for i, length in enumerate(lengths):
        length = max(int(length), 0)
        filled = min(-(-length // page), columns)
        newest = min(max(length - rows, 0) // page, filled)
        for h in range(heads):
            score = np.full(filled, -np.inf)
            at = table[i, :filled]
            there = np.flatnonzero((at >= 0) & (at < bounds.shape[0]))
            low, high = bounds[at[there], 0, h], bounds[at[there], 1, h]
            with np.errstate(all="ignore"):
                for q in query[i, max(rows - length, 0):, h * shared:(h + 1) * shared].reshape(-1, query.shape[-1]):
                    sums = (q * np.where(q >= 0, high, low)).sum(-1).astype(np.float32)
                    score[there] = np.maximum(score[there], np.where(np.isnan(sums), np.inf, sums))
            always = [c for c in range(filled) if c == 0 or c >= newest]
            others = [c for c in range(filled) if not (c == 0 or c >= newest)]
            others.sort(key=lambda c: (-score[c], c))
            kept = sorted(always + others[:max(0, min(count, filled) - len(always))])
            out[i, h, :len(kept)] = table[i, kept]
            seen[i, h] = length - page * (filled - len(kept))
    return out, seen
