"""Verification of drafted tokens in numpy, float64, one sequence at a time."""

from __future__ import annotations

import numpy as np


def distribution(logits: np.ndarray, temperature: float):
    """(probabilities, their logarithms) of a row, None where it has none."""

    x = logits.astype(np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
        return None
    x = (x - x.max()) / (temperature if temperature > 0 else 1.0)
    logs = x - np.log(np.exp(x).sum())
    return np.exp(logs), logs


def verify(logits, drafts, uniforms, probs, temperature, count):
    """logits [n + 1, V], drafts [n], uniforms [n + 1] (float32 values), probs [n, V] or None.
    Returns (tokens, accepted, logprobs, refused, margin): margin is how far the nearest decision was from its border,
    of the tests relative to the draft's probability, of the draw relative to the whole."""

    rows, vocab = logits.shape
    tokens, logprobs = np.full(rows, -1, np.int64), np.zeros(rows)
    refused, margins = not 0 <= count < rows, [(np.inf, np.inf)]
    count, left, best = min(max(count, 0), rows - 1), None, None
    for j in range(count + 1):
        dist = distribution(logits[j], temperature)
        if j == count:
            left = None if dist is None else dist[0]
            break
        x = int(drafts[j])
        if not 0 <= x < vocab:
            refused = True
            left = None if dist is None else dist[0]
            break
        if dist is None:
            break
        if temperature <= 0:
            stays = int(np.argmax(logits[j])) == x
        else:
            q = 1.0 if probs is None else float(probs[j, x])
            offer, p = float(uniforms[j]) * q, float(dist[0][x])
            stays = offer < p
            if np.isfinite(offer) and max(offer, p) > 0 and offer > 0:
                margins.append((abs(offer - p) / max(offer, p), np.inf))
        if stays:
            tokens[j], logprobs[j] = x, dist[1][x]
            continue
        if probs is None:
            left = dist[0].copy()
            left[x] = 0.0
        else:
            left = dist[0] - probs[j].astype(np.float64)
            left = np.where(left <= 0, 0.0, left)  # a NaN stays
        break
    accepted = j
    token, logprob = -1, np.nan
    if dist is not None and temperature <= 0:
        token = int(np.argmax(logits[accepted]))
    elif dist is not None and left is not None and np.isfinite(left).all():
        if not left.sum() > 0:
            left = dist[0]
        running = np.cumsum(left)
        target = float(uniforms[rows - 1]) * running[-1]
        token = int(min(np.searchsorted(running, target, side="right"), np.flatnonzero(left)[-1]))
        margins.append((np.inf, float(np.abs(running - target).min() / running[-1])) if 0 < target < running[-1] else (np.inf, np.inf))
    if token >= 0:
        logprob = dist[1][token]
    refused |= token < 0
    tokens[accepted], logprobs[accepted] = token, logprob
    return tokens, accepted, logprobs, refused, tuple(min(m[i] for m in margins) for i in range(2))
