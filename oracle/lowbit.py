"""Block-scaled low-bit formats, restated in float64 numpy (formats: include/tmhd_lowbit.h).

MXFP4 by search over its eight magnitudes, 8-bit K/V by rounding to the code's
own step, but not up to 2^128, which bf16 does not hold; scales are found from
the definition (a power of two and an inequality), not from bit fields.  Values come back as the float64 numbers
that codes and scales stand for, NaN for a block that holds an infinity or NaN.
"""

from __future__ import annotations

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mxfp4_exponent(amax: np.ndarray) -> np.ndarray:
    """floor(log2 amax) - 2, not below -125 (frexp is exact)."""
    m, e = np.frexp(amax)
    del m
    return np.maximum(np.where(amax > 0, e - 3, -125), -125)


def mxfp4_values(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(values, scale bytes [rows, K / 32]) of float rows [rows, K]."""
    rows, k = x.shape
    b = x.astype(np.float64).reshape(rows, k // 32, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    e = mxfp4_exponent(np.abs(b).max(-1))
    scale = np.ldexp(1.0, e)[..., None]
    y = np.abs(b) / scale
    # nearest magnitude; at equal distance the even code, so the lower of an
    # (even, odd) pair and the upper of an (odd, even) pair; beyond 6 stays 6
    dist = np.abs(y[..., None] - E2M1)
    odd = np.arange(8) % 2
    order = np.lexsort((np.broadcast_to(odd, dist.shape), dist), axis=-1)[..., 0]
    out = np.copysign(E2M1[order] * scale, b)
    out[bad] = np.nan
    byte = np.where(bad, 255, e + 127).astype(np.uint8)
    return out.reshape(rows, k), byte


KV_TOP = {"e4m3": 448.0, "int8": 127.0}
KV_BELOW = {256.0: 240.0, 64.0: 63.0}  # the code in front of a power of two, e4m3 and int8


def kv8_values(x: np.ndarray, fmt: str) -> tuple[np.ndarray, np.ndarray]:
    """(values, scale bytes [ceil(T / 64), H]) of K or V rows [T, H, D] packed from a block's start."""
    t, h, d = x.shape
    out = np.empty((t, h, d))
    byte = np.empty(((t + 63) // 64, h), np.uint8)
    for i in range((t + 63) // 64):
        b = x[64 * i : 64 * i + 64].astype(np.float64)
        bad = ~np.isfinite(b).all((0, 2))
        b = np.where(bad[None, :, None], 0.0, b)
        amax = np.abs(b).max((0, 2))
        e = np.full(h, -117)
        while (amax > KV_TOP[fmt] * np.ldexp(1.0, e)).any():
            e = np.where(amax > KV_TOP[fmt] * np.ldexp(1.0, e), e + 1, e)
        scale = np.ldexp(1.0, e)[None, :, None]
        y = b / scale
        if fmt == "e4m3":
            m, ex = np.frexp(np.abs(y))
            del m
            step = np.ldexp(1.0, np.maximum(ex - 1, -6) - 3)
            y = np.rint(y / step) * step
        else:
            y = np.rint(y)
        for power, code in KV_BELOW.items():
            y = np.where((np.abs(y) == power) & (power * scale == 2.0**128), np.copysign(code, y), y)
        y = y * scale
        y[:, bad] = np.nan
        out[64 * i : 64 * i + 64] = y
        byte[i] = np.where(bad, 255, e + 127)
    return out, byte


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float) -> np.ndarray:
    """softmax(q k^T scale) v in float64: q [Lq, H, D], k / v [T, H, D]."""
    out = np.empty(q.shape)
    for i in range(q.shape[1]):
        s = q[:, i].astype(np.float64) @ k[:, i].T * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        out[:, i] = (p @ v[:, i]) / p.sum(-1, keepdims=True)
    return out
