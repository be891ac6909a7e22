"""The MXFP4 oracle against the format's definition: codes by hand, the
nearest representable value by brute force, fixed points, special blocks; and
the experts against a plain per-pair evaluation."""
import numpy as np
import pytest

from oracle import mxfp4 as O


def test_code_values_by_hand():
    codes = np.arange(16, dtype=np.uint8)
    packed = (codes[0::2] | (codes[1::2] << 4)).reshape(1, 8)
    row = np.concatenate([packed, np.zeros((1, 8), np.uint8)], axis=1)
    v = O.dequantize(row, np.array([[127]], np.uint8))[0]
    assert v[:16].tolist() == [0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6]
    assert np.array_equal(O.dequantize(row, np.array([[130]], np.uint8))[0], 8 * v)
    assert np.isnan(O.dequantize(row, np.array([[255]], np.uint8))).all()
    assert O.dequantize(row, np.array([[0]], np.uint8))[0, 7] == 6 * 2.0 ** -127


def test_ties_go_to_the_even_code():
    # block maximum 6: scale 1
    v = np.array([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, -.25, -.75, -5.0] + [0] * 21, np.float32)
    q, s = O.quantize(v.reshape(1, 32))
    assert s[0, 0] == 127
    got = O.dequantize(q, s)[0]
    assert got[:11].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, -4]


def test_nearest_value_and_saturation():
    rng = np.random.default_rng(0)
    v = (rng.standard_normal((64, 96)) * np.exp(rng.standard_normal((64, 1)) * 4)).astype(np.float32)
    q, s = O.quantize(v)
    got = O.dequantize(q, s).reshape(64, 3, 32)
    b = v.astype(np.float64).reshape(64, 3, 32)
    unit = O.scale_values(s)[..., None]
    top = np.abs(b).max(axis=-1, keepdims=True)
    assert ((top / unit >= 4) & (top / unit < 8)).all()
    grid = np.concatenate([O.MAGNITUDES, -O.MAGNITUDES])
    best = np.abs(b[..., None] - grid * unit[..., None]).min(axis=-1)
    assert np.array_equal(np.abs(b - got), best)


def test_values_of_the_format_are_fixed_points():
    rng = np.random.default_rng(1)
    v = rng.standard_normal((16, 64)).astype(np.float32)
    q, s = O.quantize(v)
    again = O.quantize(O.dequantize(q, s).astype(np.float32))
    assert np.array_equal(O.dequantize(*again), O.dequantize(q, s))


@pytest.mark.parametrize("value,scale", [(0.0, 0), (2.0 ** -126, 0), (2.0 ** -149, 0),
                                         (2.0 ** -124, 1), (3.4e38, 252), (np.inf, 255),
                                         (-np.inf, 255), (np.nan, 255)])
def test_special_blocks(value, scale):
    v = np.zeros((1, 32), np.float32)
    v[0, 5] = value
    q, s = O.quantize(v)
    assert s[0, 0] == scale
    if scale == 255:
        assert not q.any()


def test_experts_against_plain_pairs():
    rng = np.random.default_rng(2)
    T, H, I, E, K = 5, 64, 32, 4, 2
    w13, s13 = O.quantize(rng.standard_normal((E, 2 * I, H)).astype(np.float32))
    w2, s2 = O.quantize(rng.standard_normal((E, H, I)).astype(np.float32))
    x = rng.standard_normal((T, H))
    w = rng.uniform(0, 1, (T, K))
    slots = np.stack([rng.permutation(E)[:K] for _ in range(T)])
    slots[2, 1] = -1
    out, bound = O.experts(x, w, slots, w13, s13, w2, s2)
    for t in range(T):
        want = np.zeros(H)
        for k in range(K):
            e = slots[t, k]
            if e >= 0:
                h = O.dequantize(w13[e], s13[e]) @ x[t]
                want += w[t, k] * (O.dequantize(w2[e], s2[e]) @ (h[:I] / (1 + np.exp(-h[:I])) * h[I:]))
        assert np.allclose(out[t], want, rtol=1e-12, atol=1e-12)
    assert (bound > 0).all()
