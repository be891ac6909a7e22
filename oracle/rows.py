"""Oracle: RMS norm with the residual's addition, SwiGLU and grouped products over
rows in 8 bits or bfloat16, in float64 on the CPU — TEST INFRASTRUCTURE ONLY.

The reference has none of these (vLLM's own operators do this work there);
parity is with the definitions (checks in ``tests/test_oracle_rows.py``).
"""
from __future__ import annotations

import numpy as np

GROUP = 128
TOP = 448.0
LEAST = 1e-10
STEP = 2.0 ** -24     # half a step of float32, relative
BF16 = 2.0 ** -8      # half a step of bfloat16, relative
TINY = 2.0 ** -133    # a step of bfloat16 near zero (and more than one of float32)


def e4m3(a: np.ndarray) -> np.ndarray:
    """The values nearest to ``a`` among those of float8_e4m3fn, ties to the
    even one, saturating at 448: four significant bits from 2^-6 up, steps of
    2^-9 below."""
    a = np.asarray(a, np.float64)
    step = np.ldexp(1.0, np.maximum(np.frexp(a)[1] - 1, -6) - 3)
    return np.clip(np.rint(a / step) * step, -TOP, TOP)


def quantize(y: np.ndarray, rel: float | np.ndarray = 0.0):
    """``(scales, low, high)`` of rows ``y [M, C]`` known to ``rel`` of each
    value: a code lies between those of the value and of its scale moved by
    that much either way (rounding is monotone)."""
    M, C = y.shape
    G = -(-C // GROUP)
    rel = np.broadcast_to(rel, y.shape)
    scales, low, high = np.zeros((M, G)), np.zeros_like(y), np.zeros_like(y)
    for g in range(G):
        at = slice(g * GROUP, (g + 1) * GROUP)
        v, r = y[:, at], rel[:, at]
        s = np.maximum(np.abs(v).max(axis=1, keepdims=True), LEAST) / TOP
        # the scale moves by its maximum's, the quotient by both and four roundings
        d = r + r.max(axis=1, keepdims=True) + 4 * STEP
        ends = e4m3(v / s * (1 - d)), e4m3(v / s * (1 + d))
        low[:, at], high[:, at] = np.minimum(*ends), np.maximum(*ends)
        scales[:, g:g + 1] = s
    return scales, low, high


def rms_norm(r: np.ndarray, weight: np.ndarray, eps: float) -> np.ndarray:
    return r / np.sqrt(np.mean(r * r, axis=1, keepdims=True) + eps) * weight


# Of the norm in float32, relative: the sum of squares adds at most 32 of a
# thread's in a row, then 4 + 3 + 15 partial ones, all positive, so it is off by
# at most 56 half steps with its products, the root by half of that and its own;
# mean, eps, root, division and the two products add six.
NORM = (28 + 6 + 2) * STEP


def silu_mul(h: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """``(y, rel)``: the SwiGLU of rows ``h [M, 2I]`` and how far float32 may
    be from it, relative: the exponential's argument is rounded twice (its error
    grows with its size), the exponential, the sum and the reciprocal are within
    a step each, three products round."""
    gate, up = np.split(h, 2, axis=1)
    with np.errstate(over="ignore"):
        y = gate / (1.0 + np.exp(-gate)) * up
    return y, (12 + 4 * np.abs(gate)) * STEP


def groups(ends, M: int) -> list[tuple[int, int]]:
    """Rows ``[first, end)`` of every group, from the definition of ends."""
    out, first = [], 0
    for e in ends:
        end = max(first, min(max(int(e), 0), M))
        out.append((first, end))
        first = end
    return out


def grouped_mm(x: np.ndarray, w: np.ndarray, ends, dot: float = 0.0):
    """``(out, bound)``: the products, zeros behind the last group, and how far
    a float32 sum may be from them: K products of which each addition is off by
    at most one step (2 half steps), plus ``dot`` of the products' sizes."""
    M, K = x.shape
    out, bound = np.zeros((M, w.shape[1])), np.zeros((M, w.shape[1]))
    for e, (a, b) in enumerate(groups(ends, M)):
        if b > a:
            out[a:b] = x[a:b] @ w[e].T
            bound[a:b] = ((K + 8) * 2 * STEP + dot) * (np.abs(x[a:b]) @ np.abs(w[e]).T)
    return out, bound


def spread(ws: np.ndarray, N: int, K: int) -> np.ndarray:
    """Block scales ``[..., ceil(N / 128), ceil(K / 128)]`` over ``[..., N, K]``."""
    return np.repeat(np.repeat(ws, GROUP, axis=-2)[..., :N, :], GROUP, axis=-1)[..., :K]
