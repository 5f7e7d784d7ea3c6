"""Draft verification by its rule, in Python integers on the CPU."""

from __future__ import annotations

import numpy as np


def _weights(w: np.ndarray) -> np.ndarray:
    w = np.where(w > 0, np.minimum(w, np.float32(1)), np.float32(0)).astype(np.float64)
    return np.rint(w * 2.0 ** 40).astype(np.int64)


def draw(weights: np.ndarray, uniform) -> int:
    """Lowest index whose prefix sum exceeds floor(uniform * total)."""

    total = int(weights.sum())
    if total == 0:
        return len(weights) - 1
    bar = min(int(np.floor(np.float64(uniform) * np.float64(total))), total - 1)
    return int(np.searchsorted(np.cumsum(weights), bar, side="right"))


def verify(target, drafts, accept, sample, query_start, width, draft_probs=None):
    """(tokens [requests, width], accepted [requests]); arrays float32 / int."""

    n = len(query_start) - 1
    tokens, accepted = np.full((n, width), -1, dtype=np.int64), np.zeros(n, dtype=np.int32)
    vocab = target.shape[1]
    for b in range(n):
        row, rows = int(query_start[b]), int(query_start[b + 1] - query_start[b])
        first, j = row - b, 0
        while j < rows - 1:
            x = int(drafts[first + j])
            if not 0 <= x < vocab:
                break
            q = draft_probs[first + j, x] if draft_probs is not None else np.float32(1)
            if not np.float32(accept[first + j]) * q < target[row + j, x]:
                break
            tokens[b, j] = x
            j += 1
        p = target[row + j]
        rest = p.copy()
        if j < rows - 1:
            if draft_probs is not None:
                rest = p - draft_probs[first + j]
            elif 0 <= int(drafts[first + j]) < vocab:
                rest[int(drafts[first + j])] = 0
        weights = _weights(rest)
        if weights.sum() == 0:
            weights = _weights(p)
        tokens[b, j] = draw(weights, sample[b])
        accepted[b] = j
    return tokens, accepted
