"""The 8-bit paged cache and its attention from their formulas, in 64 bits on the CPU.

Codes are numpy arrays [blocks, heads, block, d] of int8, or of uint8 holding
e4m3 bit patterns; scales float32 [blocks, heads].  Slow and plain on purpose.
"""

from __future__ import annotations

import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0}


def e4m3_values() -> np.ndarray:
    """Value of each e4m3 bit pattern: 1 sign, 4 exponent (bias 7) and 3
    mantissa bits; no infinities, NaN at the two all-ones patterns."""

    out = np.empty(256)
    for i in range(256):
        e, m = (i >> 3) & 15, i & 7
        v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[i] = np.nan if (i & 127) == 127 else v
        if i & 128:
            out[i] = -out[i]
    return out


_E4M3 = e4m3_values()


def code_values(codes: np.ndarray, code: str) -> np.ndarray:
    return codes.astype(np.float64) if code == "int8" else _E4M3[codes]


def half_step(value: np.ndarray, code: str) -> np.ndarray:
    """Half the distance between neighbouring codes around ``value`` (in units of the scale)."""

    if code == "int8":
        return np.full_like(value, 0.5)
    return np.maximum(np.abs(value) * 2.0 ** -4, 2.0 ** -10)


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray) -> np.ndarray:
    """x [tokens, heads, d] by [tokens, d] tables."""

    half = x.shape[-1] // 2
    x, cos, sin = x.astype(np.float64), cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
    flipped = np.concatenate((-x[..., half:], x[..., :half]), axis=-1)
    return x * cos + flipped * sin


def dequantise(codes: np.ndarray, scales: np.ndarray, code: str) -> np.ndarray:
    return code_values(codes, code) * scales.astype(np.float64)[..., None, None]


def attend(query: np.ndarray, keys: np.ndarray, values: np.ndarray, tables, requests, scale: float):
    """Attention and its magnitude sum_j p_j |v_j| and the largest scale *
    sum_d |q_d k_jd| of each row; keys and values are dequantised [blocks,
    heads, block, d], requests [(computed, queries)]."""

    tokens, hq, d = query.shape
    hkv, bs = keys.shape[1], keys.shape[2]
    out, size, reach = (np.zeros(s) for s in ((tokens, hq, d), (tokens, hq, d), (tokens, hq)))
    t = 0
    for r, (computed, n) in enumerate(requests):
        for i in range(n):
            end = computed + i + 1
            ids = np.asarray(tables[r][: -(-end // bs)])
            k = keys[ids].transpose(1, 0, 2, 3).reshape(hkv, -1, d)[:, :end]
            v = values[ids].transpose(1, 0, 2, 3).reshape(hkv, -1, d)[:, :end]
            for h in range(hq):
                g = h // (hq // hkv)
                q = query[t, h].astype(np.float64)
                s = k[g] @ q * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h] = p @ v[g]
                size[t, h] = p @ np.abs(v[g])
                reach[t, h] = (np.abs(k[g]) @ np.abs(q)).max() * scale
            t += 1
    return out, size, reach
