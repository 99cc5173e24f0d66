"""The 8-bit block cache and the head norm in numpy: codes and selections in the
float32 steps that define them, norms and attention in float64."""

from __future__ import annotations

import numpy as np

LEAST_SCALE = np.float32(2.0 ** -120)


def scale_of(amax: np.float32) -> np.float32:
    scale = np.float32(amax) / np.float32(127)
    return LEAST_SCALE if scale < LEAST_SCALE else scale


def codes_of(rows: np.ndarray, scale: np.float32) -> np.ndarray:
    with np.errstate(all="ignore"):
        product = rows.astype(np.float32) * (np.float32(1) / scale)
    return np.nan_to_num(np.clip(np.rint(product), -127, 127), nan=0.0).astype(np.int8)


def quantise(rows: np.ndarray) -> tuple[np.ndarray, np.float32]:
    """Codes and scale of one block's rows [m, D] of one head."""

    rows = rows.astype(np.float32)
    with np.errstate(all="ignore"):
        amax = np.abs(rows).max()  # NaN propagates
        scale = scale_of(amax)
    return codes_of(rows, scale), scale


def head_norm_rope(x, weight, cos, sin, positions, eps, interleaved):
    """[T, H, D] -> float64."""

    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if weight is not None:
        y = y * weight.astype(np.float64)
    if cos is None:
        return y
    c, s = (t.astype(np.float64)[positions][:, None] for t in (cos, sin))
    rot = 2 * c.shape[-1]
    out = y.copy()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = y[..., first], y[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    return out


def attention(query, keys, values, scale, visible):
    """query [L, Hq, D]; keys, values [Hkv][n, D] float64; visible [Hkv][L, n] truth values.
    Returns (out [L, Hq, D], lse [L, Hq], weighted mean magnitude of the values [L, Hq, D])."""

    length, heads, dim = query.shape
    group = heads // len(keys)
    out, size = np.zeros((length, heads, dim)), np.zeros((length, heads, dim))
    lse = np.full((length, heads), -np.inf)
    for l in range(length):
        for h in range(heads):
            seen = visible[h // group][l]
            if not seen.any():
                continue
            logits = keys[h // group][seen] @ query[l, h].astype(np.float64) * scale
            top = logits.max()
            p = np.exp(logits - top)
            lse[l, h] = top + np.log(p.sum())
            out[l, h] = p @ values[h // group][seen] / p.sum()
            size[l, h] = p @ np.abs(values[h // group][seen]) / p.sum()
    return out, lse, size


def select(query, low, high, key_scale, count, first, recent):
    """query [Hq, D]; low, high [Hkv][n, D] codes; key_scale [Hkv][n]: blocks [Hkv, count]."""

    heads = len(low)
    group = query.shape[0] // heads
    result = np.full((heads, count), -1, np.int32)
    for h in range(heads):
        n = low[h].shape[0]
        best = np.full(n, -np.inf, np.float32)
        with np.errstate(all="ignore"):
            for g in range(group):
                codes, scale = quantise(query[h * group + g][None])
                q = codes[0].astype(np.int64)
                bound = np.maximum(q * low[h].astype(np.int64), q * high[h].astype(np.int64)).sum(1)
                best = np.maximum(best, bound.astype(np.float32) * scale)  # NaN propagates
            score = best * key_scale[h].astype(np.float32)
        score = np.where(np.isnan(score), np.inf, score.astype(np.float64))  # a NaN goes before every number
        nan_first = np.where(np.isnan(best * key_scale[h]), 0, 1)
        forced = [j for j in range(n) if j < first or j >= n - recent]
        rest = sorted((j for j in range(n) if j not in set(forced)), key=lambda j: (nan_first[j], -score[j], j))
        kept = sorted(forced[:count] + rest[:max(0, count - len(forced))])
        result[h, :len(kept)] = kept
    return result
