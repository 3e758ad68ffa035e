"""Plain attention in 64 bits for the tests, and how far a result that keeps
its sums in f32 and rounds weights and outputs to the storage type may be from it."""
from __future__ import annotations

import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST_STEP = {torch.float32: 0.0, torch.float16: 2.0 ** -24, torch.bfloat16: 0.0}  # of subnormals that attention meets


def seen_keys(rows: int, first: int, keys: int, causal: bool, window: int, sinks: int) -> np.ndarray:
    """[rows, keys]: whether query i, at position first + i, sees key j."""
    position, place = first + np.arange(rows, dtype=np.int64)[:, None], np.arange(keys, dtype=np.int64)[None, :]
    if not causal:
        return np.ones((rows, keys), bool)
    seen = place <= position
    return seen & ((place > position - window) | (place < sinks)) if window else seen


def attention_rows(q, k, v, first, causal, window, sinks, scale, dtype, missing=()):
    """One sequence in float64: q [R, Hq, D], k / v [N, H, D] (numpy); query i stands at first + i; `missing` keys do not exist.
    Returns outputs [R, Hq, D], logarithms [R, Hq] and the bounds of both.  (Values that are no numbers count for nothing: the
    tests look at rows that do not see them.)

    With u the storage type's half step, d the depth and n the keys seen, a row's products are d products and sums in f32:
    a score is off by at most e = (d + 2) 2^-24 |scale| sum |q k|, and by 4 roundings of its own magnitude on the way to
    the power of two; so its weight by the factor 1 + 2 e and a little (2^-20 covers the function and second orders), and the
    normalised one by twice that.  Weights are rounded once (u), the n products are summed in f32 (n + 16 covers joins and
    rescaling), the result is rounded once (u, and half a subnormal step; a weight's subnormal rounding counts for every key)."""
    rows, heads, depth = q.shape
    shared = heads // k.shape[1] if k.shape[1] else 1
    out, logs = np.zeros((rows, heads, depth)), np.full((rows, heads), -np.inf)
    bound, log_bound = np.zeros_like(out), np.zeros_like(logs)
    u, step = HALF_STEP[dtype], SMALLEST_STEP[dtype]
    seen = seen_keys(rows, first, k.shape[0], causal, window, sinks)
    seen[:, [j for j in missing if j < k.shape[0]]] = False
    n = seen.sum(1)
    some = n > 0
    if not some.any():
        return out, logs, bound, log_bound
    for h in range(heads):
        kh, vh = k[:, h // shared], np.where(np.isfinite(v[:, h // shared]), v[:, h // shared], 0.0)
        with np.errstate(all="ignore"):
            score = np.where(seen, scale * (q[:, h] @ kh.T), -np.inf)[some]
            top = score.max(1)
            weight = np.where(seen[some], np.exp(score - top[:, None]), 0.0)
            total = weight.sum(1)
            out[some, h] = weight @ vh / total[:, None]
            logs[some, h] = top + np.log(total)
            size = np.where(seen, abs(scale) * (np.abs(q[:, h]) @ np.abs(kh).T), 0.0)[some].max(1)
            largest = np.where(seen[some], np.abs(score), 0.0).max(1)
            e = ((depth + 2) * size + 4 * largest) * 2.0 ** -24 + 2.0 ** -20
            spread = weight @ np.abs(vh) / total[:, None]
            bound[some, h] = ((u * np.abs(out[some, h]) + spread * (u + 4 * e + (n[some] + 16) * 2.0 ** -24)[:, None]) * 1.01
                              + step / 2 + n[some][:, None] * step / 2 * np.abs(vh).max())
            log_bound[some, h] = 2 * e + (n[some] + 16) * 2.0 ** -24 + 4 * 2.0 ** -24 * (np.abs(logs[some, h]) + np.abs(top))
    return out, logs, bound, log_bound


def assert_within(got: torch.Tensor, want: np.ndarray, bound: np.ndarray) -> None:
    got = got.detach().double().cpu().numpy().reshape(want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN positions differ"
    infinite = np.isinf(want)
    assert np.array_equal(got[infinite], want[infinite]), "infinities differ"
    fine = np.isfinite(want)
    assert np.isfinite(got[fine]).all(), "values that are not finite"
    off = np.abs(got[fine] - want[fine]) - bound[fine]
    if off.size and off.max() > 0:
        at = int(np.argmax(off))
        raise AssertionError(f"{int((off > 0).sum())} of {off.size} outside: got {got[fine][at]!r} want {want[fine][at]!r} bound {bound[fine][at]:.3e}")
