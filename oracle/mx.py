"""Microscaled 4-bit rows in NumPy: blocks of 32 columns with a power-of-two scale and e2m1 codes.

No counterpart in the reference; the format is the published microscaling one (e2m1 elements, e8m0 scales).  Written for
clarity: the nearest level is found by comparing distances in fp64, where every input and level is exact.
"""

from __future__ import annotations

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def quantize(x) -> tuple[np.ndarray, np.ndarray]:
    """(codes uint8 [T, P / 2], scales uint8 [T, P / 32]) of real rows [T, K], P = K rounded up to 32."""
    x = np.asarray(x, np.float64)
    T, K = x.shape
    v = np.zeros((T, -(-K // BLOCK) * BLOCK))
    v[:, :K] = x
    v = v.reshape(T, -1, BLOCK)
    bad = ~np.isfinite(v).all(axis=2)
    v = np.where(bad[..., None], 0.0, v)
    top = np.abs(v).max(axis=2)
    _, e = np.frexp(top)  # top in [2^(e-1), 2^e)
    s = np.where(top > 0, np.clip(e - 1 - 2, -127, 127), -127)
    a = np.minimum(np.abs(v) * np.exp2(-s.astype(np.float64))[..., None], 6.0)
    d = np.abs(a[..., None] - LEVELS)
    # The nearest level, of two as near the one with an even index: odd indices a hair further away.
    code = np.argmin(np.where(d == d.min(axis=-1, keepdims=True), np.arange(8) % 2, 2), axis=-1)
    code = code + np.where(np.signbit(v), 8, 0)
    code = np.where(bad[..., None], 0, code).reshape(T, -1).astype(np.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, np.where(bad, 255, s + 127).astype(np.uint8)


def dequantize(codes, scales, K: int | None = None) -> np.ndarray:
    """fp64 values of codes [..., P / 2] and scales [..., P / 32], the first K columns."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    n = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = np.where(n >= 8, -1.0, 1.0) * LEVELS[n & 7]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    v = v * np.repeat(s, BLOCK, axis=-1)
    return v if K is None else v[..., :K]
