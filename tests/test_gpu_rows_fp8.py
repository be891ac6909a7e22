"""The norms and the SwiGLU on the GPU against the float64 oracle: outputs
within what float32 steps and one rounding allow (derived in ``oracle.rows``),
codes between those of the value moved by that much either way."""
import numpy as np
import pytest
import torch

from oracle import rows as O
from wisp.integrations.vllm import rows_fp8 as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-6


def _f64(t):
    return t.detach().cpu().double().numpy()


def _bits(t):
    t = t.contiguous()
    return t.view(torch.int16 if t.element_size() == 2 else
                  torch.int32 if t.element_size() == 4 else torch.uint8)


def _randn(shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _near(got, want, rel, dtype):
    d = np.abs(_f64(got) - want)
    half = O.BF16 if dtype == BF else O.STEP
    bound = rel * np.abs(want)
    bound = bound + half * (np.abs(want) + bound) + O.TINY
    assert got.dtype == dtype
    assert np.all(d <= bound), float((d / bound).max())


def _codes(q, s, y, rel):
    """Codes and scales of values ``y`` known to ``rel``."""
    want, low, high = O.quantize(y, rel)
    rel = np.broadcast_to(rel, y.shape)
    worst = np.stack([rel[:, g * 128:(g + 1) * 128].max(axis=1) for g in range(s.shape[1])], 1)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == F32
    assert np.all(np.abs(_f64(s) - want) <= (worst + 2 * O.STEP) * want)
    got = _f64(q.float())
    bad = (got < low) | (got > high)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], low[bad][:4], high[bad][:4])


def _sum(x, res):
    """The new residual, exactly: one rounding of the exact sum."""
    return (x.double() + res.double()).to(res.dtype)


def _check_norm(x, w, eps, res):
    out, r = R.add_rms_norm(x, w, eps, res)
    both = torch.empty((x.shape[0], x.shape[1]), dtype=x.dtype, device=x.device)
    q, s, r8 = R.add_rms_norm_fp8(x, w, eps, res, out=both)
    q2, s2, _ = R.add_rms_norm_fp8(x, w, eps, res)
    if res is None:
        assert r is None and r8 is None
        v = x
    else:
        v = _sum(x, res)
        assert torch.equal(_bits(r), _bits(v)) and torch.equal(_bits(r8), _bits(v))
    y = O.rms_norm(_f64(v), _f64(w), eps)
    _near(out, y, O.NORM, x.dtype)
    assert torch.equal(_bits(both), _bits(out))
    _codes(q, s, y, O.NORM)
    assert torch.equal(_bits(q), _bits(q2)) and torch.equal(s, s2)
    return out, q, s


COLS = (1, 2, 7, 8, 16, 64, 120, 127, 128, 129, 136, 255, 256, 352, 504, 512, 513, 520, 1056, 1375,
        1376, 2048, 2056, 4096, 4104, 5000, 8192, 8193, 8200, 14336, 32767, 32768)


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("types", [(BF, BF, BF), (BF, F32, BF), (BF, BF, F32), (BF, F32, F32),
                                   (BF, None, BF), (BF, None, F32), (F32, F32, F32),
                                   (F32, None, F32)])
def test_norm_sizes(cols, types):
    xt, rt, wt = types
    rows = 5 if cols < 8192 else 3
    x = _randn((rows, cols), cols, xt)
    res = None if rt is None else _randn((rows, cols), cols + 1, rt, 3.0)
    w = (1.0 + 0.2 * _randn((cols,), cols + 2)).to(wt)
    _check_norm(x, w, EPS, res)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 15, 16, 17, 64, 1000])
@pytest.mark.parametrize("cols", [128, 96, 512, 2048])
def test_norm_rows(rows, cols):
    _check_norm(_randn((rows, cols), rows, BF), _randn((cols,), 1, BF), EPS,
                _randn((rows, cols), rows + 7, BF))


def test_norm_many_short_rows():
    x = _randn((70001, 128), 1, BF)
    w = _randn((128,), 2, BF)
    out, _ = R.add_rms_norm(x, w, EPS)
    _near(out, O.rms_norm(_f64(x), _f64(w), EPS), O.NORM, BF)


def test_norm_wide_range_of_values():
    """Rows from tiny to large, single spikes, zero rows (the scale's floor)."""
    x = _randn((24, 640), 3)
    x *= torch.exp2(torch.arange(-36, 36, 3, device=DEV).float())[:, None]
    x[3] = 0.0
    x[5, :] = 0.0
    x[5, 77] = -9.0
    x[9, 128:256] = 0.0
    for t in (F32, BF):
        _check_norm(x.to(t), _randn((640,), 4, t), 1e-5, None)
        _check_norm(x.to(t), _randn((640,), 4, t), 1e-5, _randn((24, 640), 5, t))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_infinities_and_nans(dtype):
    x = _randn((6, 384), 6, dtype)
    x[1, 5] = float("nan")
    x[2, 200] = float("inf")
    x[3, 383] = float("-inf")
    w = torch.ones(384, device=DEV, dtype=dtype)
    out, q, s = R.add_rms_norm(x, w, EPS)[0], *R.add_rms_norm_fp8(x, w, EPS)[:2]
    clean = torch.tensor([0, 4, 5], device=DEV)
    want, qw, sw = R.add_rms_norm(x[clean], w, EPS)[0], *R.add_rms_norm_fp8(x[clean], w, EPS)[:2]
    assert torch.equal(out[clean], want) and torch.equal(_bits(q)[clean], _bits(qw))
    assert torch.equal(s[clean], sw)
    assert out[1].isnan().all() and q[1].float().isnan().all()
    # an infinite mean: what is finite becomes zero, the infinity itself no number
    for r, c in ((2, 200), (3, 383)):
        assert out[r, c].isnan() and out[r].nan_to_num().abs().max() == 0
        g = c // 128
        for k in range(3):
            codes = q[r, 128 * k:128 * (k + 1)].float()
            assert codes.isnan().all() if k == g else codes.abs().max() == 0
    # a norm of finite values whose product with the weight is infinite
    w[130] = 3e38
    y = R.add_rms_norm_fp8((x[:1] * 0 + 1) * torch.linspace(0.1, 9, 384, device=DEV).to(dtype),
                           w * 4, EPS)
    bad = y[0][0].float().isnan().reshape(3, 128)
    assert bad[1].all() and not bad[0].any() and not bad[2].any()


def test_norm_strides_and_offsets():
    """Rows of a wider buffer, every alignment, transposed input, columns of
    one buffer read and written side by side."""
    base = _randn((9, 3001), 8, BF)
    res = _randn((9, 2999), 9, BF)
    w = _randn((1400,), 10, BF)
    for off in (0, 1, 3, 8, 16):
        for cols in (1376, 1375, 264):
            _check_norm(base[:, off:off + cols], w[off:off + cols], EPS, res[:, off:off + cols])
    _check_norm(base[:8, :9].t(), w[:8], EPS, None)
    _check_norm(base[:1, :512].expand(6, 512), w[:512], EPS, res[:6, :512])
    buf = _randn((7, 1024), 11, BF)
    keep = buf.clone()
    want, r = R.add_rms_norm(keep[:, :512], w[:512], EPS, res[:7, :512])
    got, r2 = R.add_rms_norm(buf[:, :512], w[:512], EPS, res[:7, :512],
                             residual_out=buf[:, 512:])
    assert r2.data_ptr() == buf[:, 512:].data_ptr() and torch.equal(buf[:, 512:], r)
    assert torch.equal(got, want) and torch.equal(buf[:, :512], keep[:, :512])


@pytest.mark.parametrize("cols", [96, 100, 2048, 6000])
def test_norm_in_place(cols):
    x, res = _randn((33, cols), 12, BF), _randn((33, cols), 13, BF)
    w = _randn((cols,), 14, BF)
    want, r = R.add_rms_norm(x, w, EPS, res)
    q, s, _ = R.add_rms_norm_fp8(x, w, EPS, res)
    a, b = x.clone(), res.clone()
    out, rr = R.add_rms_norm(a, w, EPS, b, out=a, residual_out=b)
    assert out is a and rr is b and torch.equal(a, want) and torch.equal(b, r)
    a, b = x.clone(), res.clone()
    R.add_rms_norm(a, w, EPS, b, out=b, residual_out=a)
    assert torch.equal(b, want) and torch.equal(a, r)
    a, b = x.clone(), res.clone()
    q2, s2, _ = R.add_rms_norm_fp8(a, w, EPS, b, residual_out=b)
    assert torch.equal(_bits(q), _bits(q2)) and torch.equal(s, s2) and torch.equal(b, r)
    assert torch.equal(a, x)


def test_norm_codes_are_the_quantiser_s():
    """From float32 rows, codes and scales are those of the standing quantiser
    on the norm's float32 output, but for values within a step of a border."""
    from wisp_amd import _lib
    x, w = _randn((64, 2048), 15), 1 + 0.1 * _randn((2048,), 16)
    y, _ = R.add_rms_norm(x, w, EPS)
    q, s, _ = R.add_rms_norm_fp8(x, w, EPS)
    qr = torch.empty((64, 2048), dtype=torch.uint8, device=DEV)
    sr = torch.empty((64, 16), dtype=F32, device=DEV)
    _lib.check(_lib.lib().wisp_quant_fp8_groups(y.data_ptr(), _lib.WISP_F32, 64, 2048, 128,
                                                qr.data_ptr(), sr.data_ptr(),
                                                _lib.stream_handle()), "quant")
    assert torch.equal(s, sr)
    differ = _bits(q) != qr
    a = (y.view(64, 16, 128) / s[..., None]).view(64, 2048).double()
    ends = O.e4m3(_f64(a * (1 - 4 * O.STEP))) != O.e4m3(_f64(a * (1 + 4 * O.STEP)))
    assert not (differ.cpu().numpy() & ~ends).any()


# ---------------------------------------------------------------------------
# SwiGLU
# ---------------------------------------------------------------------------


def _check_silu(h):
    q, s = R.silu_mul_fp8(h)
    assert q.shape == (h.shape[0], h.shape[1] // 2)
    y, rel = O.silu_mul(_f64(h))
    _codes(q, s, y, rel)
    return q, s


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("inter", [1, 7, 8, 100, 127, 128, 129, 136, 352, 353, 768, 1056, 14336])
@pytest.mark.parametrize("rows", [1, 3, 17, 130])
def test_silu_sizes(rows, inter, dtype):
    _check_silu(_randn((rows, 2 * inter), rows + inter, dtype, 2.0))


def test_silu_far_gates():
    """Gates to -80, where the value all but vanishes, and far positive ones."""
    h = _randn((16, 512), 20)
    h[:, :256] = torch.linspace(-80, 80, 256, device=DEV)[None]
    _check_silu(h)
    _check_silu(h.to(BF))


def test_silu_beyond_the_exponential():
    """Gates below -88: the exponential overflows and the value is zero."""
    h = torch.ones((2, 256), device=DEV)
    h[0, :128] = torch.linspace(-200, -90, 128, device=DEV)
    h[1, 3] = -1e30
    q, s = R.silu_mul_fp8(h)
    assert q[0].float().abs().max() == 0 and q[1, 3].float() == 0
    assert torch.isfinite(s).all() and torch.isfinite(q.float()).all()


def _check_silu_values(g, u, rel, low=0.0):
    """The SwiGLU of gates ``g`` and factors ``u`` (1-D) to ``rel`` of each value
    and ``low`` more: alone in its group a value is its scale's maximum, so the
    scale shows it to two roundings; once in rows of one value, once in groups
    that hold it 128 times."""
    gate = _f64(g)
    with np.errstate(over="ignore"):
        want = np.abs(gate / (1.0 + np.exp(-gate)) * _f64(u))
    assert want.min() >= 2 * O.LEAST and want.max() < 3e38
    for wide in (1, 128):
        h = torch.cat([g[:, None].expand(-1, wide), u[:, None].expand(-1, wide)], dim=1)
        q, s = R.silu_mul_fp8(h)
        off = np.abs(_f64(s)[:, 0] * 448 - want) / (rel * want + low + 2 * O.STEP * want)
        assert off.max() <= 1, (float(off.max()), float(g[int(off.argmax())]))
        sign = np.sign(_f64(g) * _f64(u))[:, None]
        assert np.array_equal(_f64(q.float()), np.broadcast_to(448.0 * sign, q.shape))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_silu_largest_gates(dtype):
    """Gates up to the largest finite value: the SiLU is the gate itself, and with a
    small factor the value is finite."""
    top = float(torch.finfo(dtype).max)
    g = torch.tensor([129.0, 1e4, 1e30, 2.3e38, 2.36e38, 2.37e38, 2.5e38, 3e38, top] * 4,
                     device=DEV).to(dtype)
    u = torch.tensor([1e-3, -1e-3, 0.5, 2.0 ** -126], device=DEV).to(dtype).repeat_interleave(9)
    keep = (g.double() * u.double()).abs() > 1e-9
    # the sigmoid is 1, its reciprocal within a step (two half ones), two products
    _check_silu_values(g[keep], u[keep], 4 * O.STEP)
    # an infinite gate: codes that are no numbers, and the largest value's scale
    h = _randn((3, 512), 23, dtype)
    h[1, 130] = float("inf")
    q, s = R.silu_mul_fp8(h)
    assert q[1, 128:].float().isnan().all() and bool(s[1, 1] == float("inf"))
    h[1, 130] = top
    h[1, 386] = 1.0
    q, s = R.silu_mul_fp8(h)
    assert bool(s[1, 1] == torch.tensor(top) / 448) and q[1, 130].float() == 448
    assert torch.isfinite(q.float()).all() and torch.isfinite(s).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_silu_to_some_half_steps(dtype):
    """Ordinary gates to -87: an exponential within a step (two half ones), the product
    with what its exponent's rounding left, the sum, the reciprocal within a step, two
    products: seven half steps at every gate, and one for what those leave out."""
    g = torch.linspace(-87, 87, 4001, device=DEV).to(dtype)
    g = g[g != 0]
    u = torch.exp2(-torch.floor(torch.log2(g.double().abs() / (1 + torch.exp(-g.double())))))
    _check_silu_values(g, u.to(dtype), 8 * O.STEP)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_silu_gates_to_the_end_of_float32(dtype):
    """Gates whose SiLU is at the lower end of float32, with factors that bring the value
    back: to the last of its subnormal numbers (seven half steps as above, and half a
    subnormal step of the SiLU, twice for the product before it)."""
    g = torch.linspace(-100, -80, 2001, device=DEV).to(dtype)
    u = torch.full_like(g, 2.0 ** 126)
    _check_silu_values(g, u, 8 * O.STEP, 2 * 2.0 ** -150 * 2.0 ** 126)
    # beyond: nothing is left, whatever the factor
    h = torch.full((4, 256), 2.0 ** 126, device=DEV, dtype=dtype)
    h[0, :128], h[1, :128], h[2, :128] = -128, -1e30, -float(torch.finfo(dtype).max)
    h[3, :128] = torch.linspace(-300, -115, 128, device=DEV)
    q, s = R.silu_mul_fp8(h)
    # (the quotient of the host: on the device torch multiplies by the scalar's reciprocal)
    assert not q.float().any() and bool((s.cpu() == torch.tensor(1e-10) / 448).all())
    # beside them what is no number: -inf / (1 + inf) and a NaN, in their groups only
    h = torch.cat([h, h], dim=1).view(4, 2, 2, 128).transpose(1, 2).reshape(4, 512)
    want = R.silu_mul_fp8(h)
    h[1, 130], h[2, 5] = -float("inf"), float("nan")
    got = R.silu_mul_fp8(h)
    for bits, clean in ((_bits(got[0]).view(4, 2, 128), _bits(want[0]).view(4, 2, 128)),
                        (_bits(got[1]), _bits(want[1]))):
        same = (bits == clean).view(4, 2, -1).all(dim=2)
        assert same.tolist() == [[True, True], [True, False], [False, True], [True, True]]
    assert got[0][1, 128:].float().isnan().all() and got[0][2, :128].float().isnan().all()


def test_silu_infinities_and_nans():
    h = _randn((5, 768), 21)
    h[0, 2], h[1, 384 + 130], h[2, 300] = float("nan"), float("inf"), float("inf")
    q, s = R.silu_mul_fp8(h)
    bad = q.float().isnan().reshape(5, 3, 128)
    assert bad[0, 0].all() and bad[1, 1].all() and bad[2, 2].all()
    assert int(bad.sum()) == 3 * 128


def test_silu_strides():
    h = _randn((11, 1500), 22, BF)
    for off, inter in ((0, 352), (4, 352), (1, 200), (8, 256)):
        part = h[:, off:off + 2 * inter]
        q, s = _check_silu(part)
        qc, sc = R.silu_mul_fp8(part.contiguous())
        assert torch.equal(_bits(q), _bits(qc)) and torch.equal(s, sc)
    _check_silu(h[:10, :6].t())


# ---------------------------------------------------------------------------
# Uses
# ---------------------------------------------------------------------------


def test_empty():
    w = torch.ones(64, device=DEV, dtype=BF)
    out, r = R.add_rms_norm(torch.empty((0, 64), device=DEV, dtype=BF), w, EPS,
                            torch.empty((0, 64), device=DEV, dtype=BF))
    assert out.shape == r.shape == (0, 64)
    q, s, r = R.add_rms_norm_fp8(torch.empty((3, 0), device=DEV, dtype=BF), w[:0])
    assert q.shape == (3, 0) and s.shape == (3, 0) and r is None
    q, s = R.silu_mul_fp8(torch.empty((0, 64), device=DEV, dtype=BF))
    assert q.shape == (0, 32) and s.shape == (0, 1)
    q, s = R.silu_mul_fp8(torch.empty((4, 0), device=DEV, dtype=BF))
    assert q.shape == (4, 0)


def test_norm_rows_beyond_32_bits():
    """Row offsets past 2^31 values."""
    cols, rows = 32768, 65540
    x = torch.zeros((rows, cols), device=DEV, dtype=BF)
    x[-3:] = _randn((3, cols), 30, BF)
    w = _randn((cols,), 31, BF)
    out, _ = R.add_rms_norm(x, w, EPS)
    q, s, _ = R.add_rms_norm_fp8(x, w, EPS)
    want, _ = R.add_rms_norm(x[-3:].clone(), w, EPS)
    wq, ws, _ = R.add_rms_norm_fp8(x[-3:].clone(), w, EPS)
    assert torch.equal(out[-3:], want) and not out[:-3].any()
    assert torch.equal(_bits(q[-3:]), _bits(wq)) and torch.equal(s[-3:], ws)


def test_norm_in_a_graph_and_on_streams():
    x, res, w = _randn((40, 1056), 32, BF), _randn((40, 1056), 33, BF), _randn((1056,), 34, BF)
    h = _randn((40, 704), 35, BF)
    want = (*R.add_rms_norm_fp8(x, w, EPS, res), *R.silu_mul_fp8(h))
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = (*R.add_rms_norm_fp8(x, w, EPS, res), *R.silu_mul_fp8(h))
    for _ in range(3):
        for t in got:
            _bits(t).zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(got, want))
        R.add_rms_norm(x, w, EPS)
    with torch.cuda.stream(side):
        again = (*R.add_rms_norm_fp8(x, w, EPS, res), *R.silu_mul_fp8(h))
    side.synchronize()
    assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(again, want))


def test_refusals():
    x, w = _randn((4, 64), 40, BF), _randn((64,), 41, BF)
    res = x.clone()
    for bad in (lambda: R.add_rms_norm(x[0], w), lambda: R.add_rms_norm(x, w[:63]),
                lambda: R.add_rms_norm(x, w, EPS, res[:, :32]),
                lambda: R.add_rms_norm(x, w, EPS, res.cpu()), lambda: R.add_rms_norm(x, w.cpu()),
                lambda: R.add_rms_norm(x, w, EPS, residual_out=res),
                lambda: R.add_rms_norm(x, w, EPS, res, residual_out=res.float()),
                lambda: R.add_rms_norm(x, w, EPS, res, residual_out=res[:3]),
                lambda: R.add_rms_norm(x, w, EPS, res, residual_out=res[:1].expand(4, 64)),
                lambda: R.add_rms_norm(x, w, out=x.float()),
                lambda: R.add_rms_norm(x[:, :32], w[:32], out=x[:, :32]),
                lambda: R.add_rms_norm(x, w, EPS, res, out=x, residual_out=x),
                lambda: R.add_rms_norm(x[:3], w, out=x[1:]),
                lambda: R.silu_mul_fp8(x[:, :63]), lambda: R.silu_mul_fp8(x[0])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: R.add_rms_norm(x.half(), w.half()), lambda: R.add_rms_norm(x.float(), w),
                lambda: R.add_rms_norm(x, w.half()), lambda: R.silu_mul_fp8(x.half()),
                lambda: R.add_rms_norm(x[:, :1].expand(4, 40000), w[:1].expand(40000)),
                lambda: R.add_rms_norm(x[:, :1].expand(4, 2 ** 32 + 64),
                                       w[:1].expand(2 ** 32 + 64)),
                lambda: R.silu_mul_fp8(x[:, :1].expand(4, 2 ** 33 + 128))):
        with pytest.raises(NotImplementedError):
            bad()
