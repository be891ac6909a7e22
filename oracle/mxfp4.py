"""Oracle: MXFP4 quantisation and experts over MXFP4 weights, in float64 on the
CPU — TEST INFRASTRUCTURE ONLY.

The format is the OCP microscaling one: E2M1 codes in blocks of 32 along a row
with an E8M0 scale byte each.  The reference has no such path; parity is with
the format's definition (checks in ``tests/test_oracle_mxfp4.py``).
"""
from __future__ import annotations

import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def scale_values(scales: np.ndarray) -> np.ndarray:
    s = scales.astype(np.int64)
    return np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))


def dequantize(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """float64 values of codes ``[..., C/2]`` and scales ``[..., C/32]``."""
    c = np.stack([codes & 15, codes >> 4], axis=-1).reshape(*codes.shape[:-1], -1)
    v = np.where(c >= 8, -MAGNITUDES[c & 7], MAGNITUDES[c & 7])
    return v * np.repeat(scale_values(scales), BLOCK, axis=-1)


def quantize(w: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """``w [..., C]`` float32 -> (codes, scales): by search over the eight
    magnitudes, of two equally near ones the even code."""
    b = w.astype(np.float64).reshape(*w.shape[:-1], -1, BLOCK)
    bad = ~np.isfinite(b).all(axis=-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(axis=-1)
    e = np.where(top > 0, np.frexp(top)[1] - 3, -127)
    e = np.clip(e, -127, 127)
    a = np.abs(b) / np.ldexp(1.0, e)[..., None]
    dist = np.abs(a[..., None] - MAGNITUDES)
    dist[..., 1::2] *= 1.0 + 1e-15  # an odd code has to be strictly nearer
    code = dist.argmin(axis=-1) + 8 * np.signbit(b)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    code = code.reshape(*w.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def experts(x, topk_w, slots, w13, s13, w2, s2):
    """``(out, bound)`` float64 ``[T, H]``: the SwiGLU experts' weighted sum
    without any rounding, and how far a result may be from it whose sums are
    float32 and whose act and output are rounded to bf16 (half a step, 2^-8 of
    the value, each).  Sums of n products in float32, in any order and with
    each addition off by at most one step, are off by n 2^-23 of the sum of
    the magnitudes."""
    x = np.asarray(x, np.float64)
    T, H = x.shape
    I = 2 * w2.shape[2]
    half, step = 2.0 ** -8, 2.0 ** -23
    out, bound = np.zeros((T, H)), np.zeros((T, H))
    for e in range(w13.shape[0]):
        t, k = np.nonzero(np.asarray(slots) == e)
        if t.size == 0:
            continue
        a, b = dequantize(w13[e], s13[e]), dequantize(w2[e], s2[e])
        h = x[t] @ a.T
        dh = (H + 4) * step * (np.abs(x[t]) @ np.abs(a).T)
        g, u, dg, du = h[:, :I], h[:, I:], dh[:, :I], dh[:, I:]
        with np.errstate(over="ignore"):
            silu = g / (1.0 + np.exp(-g))
        act = silu * u
        # |silu'| <= 1.1; 16 steps for the exponential, the division and the products
        dact = 1.1 * dg * (np.abs(u) + du) + np.abs(silu) * du + 16 * step * np.abs(act)
        dact = dact + half * (np.abs(act) + dact) + 2.0 ** -133
        y, mag = act @ b.T, np.abs(act) @ np.abs(b).T
        dy = (np.abs(b) @ dact.T).T + (I + 4) * step * (mag + (np.abs(b) @ dact.T).T)
        w = np.asarray(topk_w, np.float64)[t, k][:, None]
        np.add.at(out, t, w * y)
        np.add.at(bound, t, np.abs(w) * (dy + slots.shape[1] * step * (mag + dy)))
    return out, bound + half * (np.abs(out) + bound) + 2.0 ** -133
