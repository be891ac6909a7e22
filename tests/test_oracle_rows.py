"""The oracle of the norms, the SwiGLU and the grouped products against their
definitions and torch's own float64 and e4m3 arithmetic."""
import numpy as np
import torch

from oracle import rows as O


def test_e4m3_is_torch_s_cast():
    bits = np.arange(0, 0x7f800000, 40961, dtype=np.int64).astype(np.uint32)
    v = np.concatenate([bits.view(np.float32), -bits.view(np.float32)])
    v = v[np.abs(v) <= 448]
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.e4m3(v), want)
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    codes = np.unique(codes[np.isfinite(codes)])
    assert np.array_equal(O.e4m3(codes), codes)
    # half way between two codes: the even one, which torch's cast takes too
    mid = (codes[1:] + codes[:-1]) / 2
    assert np.array_equal(O.e4m3(mid), torch.from_numpy(mid.astype(np.float32)).to(
        torch.float8_e4m3fn).double().numpy())
    assert np.array_equal(O.e4m3(np.array([449.0, 1e30, -1e30])), [448.0, 448.0, -448.0])


def test_quantize():
    r = np.random.RandomState(0)
    y = r.randn(5, 300) * np.exp(3 * r.randn(5, 1))
    y[3, 128:256] = 0
    s, low, high = O.quantize(y)
    assert s.shape == (5, 3) and np.all(low <= high)
    for g in range(3):
        part = y[:, 128 * g:128 * (g + 1)]
        assert np.allclose(s[:, g], np.maximum(np.abs(part).max(1), 1e-10) / 448, rtol=1e-15)
        back = low[:, 128 * g:128 * (g + 1)] * s[:, g:g + 1]
        # half a step: 2^-4 of the value, 2^-10 of the scale near zero
        assert np.all(np.abs(back - part) <= 2.0 ** -4 * np.abs(part) * (1 + 1e-6)
                      + 2.0 ** -10 * s[:, g:g + 1] + 1e-5 * np.abs(part))
    assert s[3, 1] == 1e-10 / 448
    wide = O.quantize(y, 0.1)
    assert np.all(wide[1] <= low) and np.all(high <= wide[2])


def test_norm_and_silu():
    r = np.random.RandomState(1)
    x, w = r.randn(4, 50), r.randn(50)
    want = torch.nn.functional.rms_norm(torch.from_numpy(x), (50,), torch.from_numpy(w), 1e-6)
    assert np.allclose(O.rms_norm(x, w, 1e-6), want.numpy(), rtol=1e-13)
    h = r.randn(4, 60) * 5
    y, rel = O.silu_mul(h)
    t = torch.from_numpy(h)
    want = torch.nn.functional.silu(t[:, :30]) * t[:, 30:]
    assert np.allclose(y, want.numpy(), rtol=1e-13) and rel.shape == y.shape


def test_groups():
    assert O.groups([2, 2, 7], 9) == [(0, 2), (2, 2), (2, 7)]
    assert O.groups([5, 3, 40, 6], 9) == [(0, 5), (5, 5), (5, 9), (9, 9)]
    assert O.groups([-4, 2], 9) == [(0, 0), (0, 2)]


def test_grouped_mm():
    r = np.random.RandomState(2)
    x, w = r.randn(9, 16), r.randn(3, 5, 16)
    out, bound = O.grouped_mm(x, w, [2, 2, 7])
    for i in range(9):
        e = 0 if i < 2 else 2
        want = w[e] @ x[i] if i < 7 else np.zeros(5)
        assert np.allclose(out[i], want, rtol=1e-13)
    assert not bound[7:].any() and (bound[:7] > 0).all()


def test_spread():
    ws = np.arange(6.0).reshape(2, 3)
    v = O.spread(ws, 130, 257)
    assert v.shape == (130, 257) and v[127, 127] == 0 and v[128, 128] == 4 and v[129, 256] == 5
