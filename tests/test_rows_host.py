"""Refusals of the norms, the SwiGLU and the grouped products: decided on the
host, before any device call, so they are checked without a GPU."""
import pytest
import torch

from wisp.integrations.vllm import grouped_mm as G
from wisp.integrations.vllm import rows_fp8 as R
from wisp_amd import _lib

OK, INVALID, UNSUPPORTED = _lib.WISP_OK, _lib.WISP_ERR_INVALID, _lib.WISP_ERR_UNSUPPORTED
F32, BF16, FP8 = _lib.WISP_F32, _lib.WISP_BF16, _lib.WISP_FP8_E4M3
P = 1 << 20  # an aligned address that is never read


def _norm(lib, x=P, dtype=BF16, rows=4, cols=64, res=None, rdt=BF16, res_out=None, w=P, wdt=BF16,
          out=P, q=None, s=None):
    return lib.wisp_add_rms_norm(x, dtype, rows, cols, 64, res, rdt, 64, res_out, 64, w, wdt, 1e-6,
                                 out, q, s, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(rows=0), OK), (dict(cols=0), OK), (dict(rows=-1), INVALID), (dict(cols=-8), INVALID),
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(out=None), INVALID),
    (dict(out=None, q=P), INVALID), (dict(res=P), INVALID), (dict(dtype=FP8), UNSUPPORTED),
    (dict(wdt=FP8), UNSUPPORTED), (dict(dtype=F32, wdt=BF16), UNSUPPORTED),
    (dict(res=P, res_out=P, rdt=FP8), UNSUPPORTED),
    (dict(dtype=F32, wdt=F32, res=P, res_out=P, rdt=BF16), UNSUPPORTED),
    (dict(cols=32769), UNSUPPORTED), (dict(rows=1 << 40), UNSUPPORTED),
])
def test_norm_arguments(hiplib, kw, rc):
    assert _norm(hiplib, **kw) == rc
    if rc != OK:
        assert hiplib.wisp_last_error()


@pytest.mark.parametrize("kw,rc", [
    (dict(rows=0), OK), (dict(inter=0), OK), (dict(rows=-1), INVALID), (dict(inter=-1), INVALID),
    (dict(dtype=FP8), INVALID), (dict(h=None), INVALID), (dict(q=None), INVALID),
    (dict(s=None), INVALID), (dict(rows=1 << 40), UNSUPPORTED),
    (dict(rows=1 << 28, inter=2 ** 31 - 1), UNSUPPORTED),
])
def test_silu_arguments(hiplib, kw, rc):
    a = dict(h=P, dtype=BF16, rows=4, inter=64, q=P, s=P)
    a.update(kw)
    assert hiplib.wisp_silu_mul_fp8(a["h"], a["dtype"], a["rows"], a["inter"], 128, a["q"], a["s"],
                                    None) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(M=0), OK), (dict(N=0), OK), (dict(E=0), INVALID), (dict(M=-1), INVALID),
    (dict(N=-1), INVALID), (dict(K=0), INVALID), (dict(x=None), INVALID), (dict(w=None), INVALID),
    (dict(ends=None), INVALID), (dict(out=None), INVALID), (dict(x_ld=56), INVALID),
    (dict(w_ld=56), INVALID), (dict(ws=-64), INVALID), (dict(E=513), UNSUPPORTED),
    (dict(K=60), UNSUPPORTED), (dict(x=P + 8), UNSUPPORTED), (dict(w=P + 2), UNSUPPORTED),
    (dict(x_ld=68), UNSUPPORTED), (dict(w_ld=68), UNSUPPORTED), (dict(ws=4100), UNSUPPORTED),
    (dict(N=1 << 24), UNSUPPORTED), (dict(x_ld=1 << 21), UNSUPPORTED), (dict(dt=FP8), INVALID),
    (dict(N=1 << 21), UNSUPPORTED), (dict(w_ld=1 << 23), UNSUPPORTED),
    (dict(N=2 ** 31 - 1, w_ld=1 << 61), UNSUPPORTED), (dict(x_ld=1 << 61), UNSUPPORTED),
    (dict(w_ld=1 << 22, N=256), UNSUPPORTED),
])
def test_grouped_arguments(hiplib, kw, rc):
    a = dict(x=P, x_ld=64, w=P, ws=4096, w_ld=64, ends=P, E=2, M=4, N=64, K=64, out=P, dt=BF16)
    a.update(kw)
    assert hiplib.wisp_grouped_mm(a["x"], a["x_ld"], a["w"], a["ws"], a["w_ld"], a["ends"], a["E"],
                                  a["M"], a["N"], a["K"], a["out"], a["dt"], 0, None) == rc
    if rc != OK:
        assert hiplib.wisp_last_error()


@pytest.mark.parametrize("kw,rc", [
    (dict(M=0), OK), (dict(N=0), OK), (dict(E=0), INVALID), (dict(K=0), INVALID),
    (dict(q=None), INVALID), (dict(s=None), INVALID), (dict(w=None), INVALID),
    (dict(ws=None), INVALID), (dict(ends=None), INVALID), (dict(out=None), INVALID),
    (dict(q_ld=128), INVALID), (dict(w_ld=128), INVALID), (dict(s_ld=1), INVALID),
    (dict(wst=-1), INVALID), (dict(wsst=-1), INVALID), (dict(E=513), UNSUPPORTED),
    (dict(K=136), UNSUPPORTED), (dict(q=P + 8), UNSUPPORTED), (dict(w=P + 8), UNSUPPORTED),
    (dict(q_ld=152), UNSUPPORTED), (dict(w_ld=152), UNSUPPORTED), (dict(wst=1032), UNSUPPORTED),
    (dict(s_ld=1 << 20), UNSUPPORTED), (dict(q_ld=1 << 22), UNSUPPORTED),
    (dict(N=1 << 24), UNSUPPORTED), (dict(N=1 << 21), UNSUPPORTED),
    (dict(w_ld=1 << 24), UNSUPPORTED), (dict(w_ld=1 << 23, N=256), UNSUPPORTED),
])
def test_grouped_fp8_arguments(hiplib, kw, rc):
    a = dict(q=P, q_ld=144, s=P, s_ld=2, w=P, wst=64 * 144, w_ld=144, ws=P, wsst=2, ends=P, E=2,
             M=4, N=64, K=144, out=P)
    a.update(kw)
    assert hiplib.wisp_grouped_mm_fp8(
        a["q"], a["q_ld"], a["s"], a["s_ld"], a["w"], a["wst"], a["w_ld"], a["ws"], a["wsst"],
        a["ends"], a["E"], a["M"], a["N"], a["K"], a["out"], 0, None) == rc


def test_host_tensors_are_refused():
    x, w = torch.zeros((2, 64)), torch.zeros(64)
    w3, ends = torch.zeros((1, 8, 64)), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: R.add_rms_norm(x, w), lambda: R.add_rms_norm_fp8(x, w),
                 lambda: R.silu_mul_fp8(x), lambda: G.grouped_mm(x, w3, ends),
                 lambda: G.grouped_mm_fp8(x, x, w3, w3, ends)):
        with pytest.raises(ValueError, match="device tensors"):
            call()


def test_overlaps():
    """Which outputs share bytes with another tensor of the call."""
    b = torch.zeros(10, 64)
    apart = [(b[:, :32], b[:, 32:]), (b[:5], b[5:]), (b[:, 8:16], b[1:, 32:40]),
             (b[:, :32], b[2:, 32:]), (b[:1, :32], b[:, 32:])]
    meet = [(b[:, :33], b[:, 32:]), (b[:6], b[5:]), (b[:, :32], b[1:, :32]), (b[:1], b[:, :3]),
            (b, b), (b[:, 31:], b[1:, :32])]
    for x, y in apart:
        assert not R._overlap(x, y) and not R._overlap(y, x)
        R._check_apart("out", x, ((y, True), (None, False)))
    for x, y in meet:
        assert R._overlap(x, y) and R._overlap(y, x)
        with pytest.raises(ValueError, match="overlaps"):
            R._check_apart("out", x, ((y, False),))
    R._check_apart("out", b, ((b, True),))
    R._check_apart("out", b[:0], ((b, False),))
    with pytest.raises(ValueError, match="overlaps"):
        R._check_apart("out", b, ((b.view(torch.int32), True),))


@pytest.mark.parametrize("kw,kernel", [
    (dict(), _lib.WISP_GROUPED_FEW), (dict(M=0), -1), (dict(N=0), -1), (dict(E=0), -1),
    (dict(E=513), -1), (dict(K=0), -1), (dict(K=60), -1), (dict(fp8=1, K=136), -1),
    (dict(dt=FP8), -1), (dict(fp8=1, dt=F32), -1), (dict(N=1 << 21), -1), (dict(K=1 << 21), -1),
    (dict(M=8192 * 8, E=128, N=1536, K=2048), _lib.WISP_GROUPED_LARGE_192),
    (dict(M=64, E=128, N=1536, K=2048), _lib.WISP_GROUPED_FEW),
    (dict(M=256, E=128, N=1536, K=2048, fp8=1), _lib.WISP_GROUPED_TILE_256),
    (dict(M=4000, E=8, N=28672, K=4096, fp8=1), _lib.WISP_GROUPED_LARGE_256),
    (dict(M=4000, E=8, N=28667, K=4096, fp8=1),
     _lib.WISP_GROUPED_TILE_256 | _lib.WISP_GROUPED_NARROW),
])
def test_the_kernel_of_a_call(hiplib, kw, kernel):
    a = dict(fp8=0, E=2, M=4, N=64, K=64, dt=BF16)
    a.update(kw)
    assert hiplib.wisp_grouped_mm_kernel(a["fp8"], a["E"], a["M"], a["N"], a["K"], P,
                                         a["dt"]) == kernel


@pytest.mark.parametrize("fp8,E,M,N,K", [(0, 128, 65536, 1536, 2048), (1, 8, 4000, 28672, 4096),
                                         (0, 4, 400, 264, 256), (1, 4, 400, 264, 256),
                                         (0, 24, 2400, 1800, 200)])
def test_outputs_between_two_dwords_are_stored_one_by_one(hiplib, fp8, E, M, N, K):
    """8- and 16-byte stores go to whole dwords: a bfloat16 output at an odd element takes
    none, one at an even element the same kernel as an aligned one."""
    def kernel(at, dt=BF16):
        return hiplib.wisp_grouped_mm_kernel(fp8, E, M, N, K, P + at, dt)

    assert kernel(0) == kernel(4) == kernel(8) and not kernel(0) & _lib.WISP_GROUPED_NARROW
    for at in (2, 6, 14):
        assert kernel(at) & _lib.WISP_GROUPED_NARROW
        assert kernel(at) & ~_lib.WISP_GROUPED_NARROW in (
            _lib.WISP_GROUPED_TILE_64, _lib.WISP_GROUPED_TILE_128, _lib.WISP_GROUPED_TILE_256)
    if not fp8:
        assert kernel(4, F32) == kernel(0, F32)


@pytest.mark.parametrize("elements", [1 << 50, 1 << 60, 1 << 61, 1 << 62, (1 << 63) - 8])
def test_strides_that_no_address_counts(hiplib, elements):
    """Strides whose bytes, or those of 512 experts, pass 64 bits are refused as any that
    are too large."""
    for x_ld, ws, w_ld in ((elements, 4096, 64), (64, elements, 64), (64, 4096, elements)):
        assert hiplib.wisp_grouped_mm(P, x_ld, P, ws, w_ld, P, 2, 4, 64, 64, P, BF16, 0,
                                      None) == UNSUPPORTED
        assert hiplib.wisp_grouped_mm_fp8(P, x_ld, P, 1, P, ws, w_ld, P, 1, P, 2, 4, 64, 64, P,
                                          0, None) == UNSUPPORTED
    for s_ld, ws in ((elements, 1), (1, elements)):
        assert hiplib.wisp_grouped_mm_fp8(P, 64, P, s_ld, P, 4096, 64, P, ws, P, 2, 4, 64, 64, P,
                                          0, None) == UNSUPPORTED
