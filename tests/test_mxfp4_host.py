"""Refusals of the MXFP4 entry points: decided on the host, before any device
call, so they are checked without a GPU."""
import ctypes as C

import pytest
import torch

from wisp.integrations.vllm import fused_moe_mxfp4 as mx
from wisp_amd import _lib

OK, INVALID, UNSUPPORTED = _lib.WISP_OK, _lib.WISP_ERR_INVALID, _lib.WISP_ERR_UNSUPPORTED
P = 1 << 20  # an aligned address that is never read


def _quant(lib, x=P, dtype=_lib.WISP_BF16, rows=4, cols=64, codes=P, scales=P):
    return lib.wisp_quant_mxfp4(x, dtype, rows, cols, codes, scales, None)


def _dequant(lib, codes=P, scales=P, rows=4, cols=64, out=P, dtype=_lib.WISP_BF16):
    return lib.wisp_dequant_mxfp4(codes, scales, rows, cols, out, dtype, None)


@pytest.mark.parametrize("call", [_quant, _dequant])
@pytest.mark.parametrize("kw,rc", [
    (dict(rows=0), OK), (dict(cols=0), OK), (dict(rows=-1), INVALID), (dict(cols=-32), INVALID),
    (dict(cols=48), UNSUPPORTED), (dict(dtype=_lib.WISP_FP8_E4M3), INVALID),
    (dict(codes=None), INVALID), (dict(scales=None), INVALID), (dict(codes=P + 2), UNSUPPORTED),
    (dict(rows=1 << 60, cols=32), UNSUPPORTED),
])
def test_matrix_arguments(hiplib, call, kw, rc):
    assert call(hiplib, **kw) == rc


def test_matrix_wide_side(hiplib):
    assert _quant(hiplib, x=None) == INVALID
    assert _quant(hiplib, x=P + 8) == UNSUPPORTED
    assert _dequant(hiplib, out=None) == INVALID
    assert _dequant(hiplib, out=P + 4) == UNSUPPORTED


def _experts(lib, T=2, H=64, I=32, K=2, nslots=4, w13s=None, s13s=None, w2s=None, s2s=None, x=P,
             w=P, slots=P, w13=P, work=P, work_bytes=1 << 20, act=P, out=P):
    n = max(H * I, 0)
    return lib.wisp_moe_experts_mxfp4(
        x, T, H, I, K, w, slots, nslots, w13, n if w13s is None else w13s, P,
        n // 16 if s13s is None else s13s, P, n // 2 if w2s is None else w2s, P,
        n // 32 if s2s is None else s2s, act, out, work, work_bytes, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(T=0), OK), (dict(T=-1), INVALID), (dict(nslots=0), INVALID), (dict(K=0), UNSUPPORTED),
    (dict(K=65), UNSUPPORTED), (dict(H=48), UNSUPPORTED), (dict(I=16), UNSUPPORTED),
    (dict(H=0), UNSUPPORTED), (dict(H=1 << 16, I=1 << 15), UNSUPPORTED),
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(slots=None), INVALID),
    (dict(w13=None), INVALID), (dict(act=None), INVALID), (dict(out=None), INVALID),
    (dict(x=P + 2), UNSUPPORTED), (dict(out=P + 8), UNSUPPORTED), (dict(w13=P + 4), UNSUPPORTED),
    (dict(w13s=64 * 32 + 8), UNSUPPORTED), (dict(w13s=64 * 32 - 16), INVALID),
    (dict(w2s=64 * 16 - 16), INVALID), (dict(s13s=64), INVALID), (dict(s2s=32), INVALID),
    (dict(s13s=130), UNSUPPORTED), (dict(s2s=66), UNSUPPORTED),
    (dict(work=None), INVALID), (dict(work=P + 16), INVALID), (dict(work_bytes=64), INVALID),
    (dict(T=1 << 26, K=64), INVALID),
])
def test_experts_arguments(hiplib, kw, rc):
    assert _experts(hiplib, **kw) == rc
    if rc != OK:
        assert hiplib.wisp_last_error()


@pytest.mark.parametrize("kw", [dict(logits=None), dict(dtype=_lib.WISP_FP8_E4M3), dict(K=5),
                                dict(w=None), dict(ids=None), dict(E=513)])
def test_layer_arguments(hiplib, kw):
    a = dict(logits=P, dtype=_lib.WISP_F32, E=4, K=2, w=P, ids=P)
    a.update(kw)
    n = 64 * 32
    assert hiplib.wisp_moe_layer_mxfp4(
        P, a["logits"], a["dtype"], 2, 64, 32, a["E"], a["K"], 1, a["w"], a["ids"], P, n, P,
        n // 16, P, n // 2, P, n // 32, P, P, P, 1 << 20, None) == INVALID


def _desc(**kw):
    H, I, E = 64, 32, 4
    n = H * I
    d = _lib.LayerDesc()
    d.struct_bytes = C.sizeof(_lib.LayerDesc)
    d.num_experts, d.cap, d.hidden, d.inter = E, 2, H, I
    d.dtype, d.mode = _lib.WISP_MXFP4, _lib.WISP_MODE_PAGED
    d.w13_elems, d.w2_elems, d.s13_elems, d.s2_elems = n, n // 2, n // 16, n // 32
    for part in ("w13", "w2", "s13", "s2"):
        for side in ("scratch_", "master_"):
            setattr(d, side + part, P)
            setattr(d, side + part + "_stride", 4096)
    d.expert_map = d.slot_to_expert = d.lru_tick = d.counters = P
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [
    dict(w13_elems=2 * 64 * 32), dict(w2_elems=64 * 32), dict(s13_elems=64), dict(s2_elems=32),
    dict(hidden=48), dict(inter=16), dict(hidden=0), dict(scratch_s13=None), dict(master_s2=None),
    dict(scratch_s13_stride=64), dict(master_w13_stride=1024), dict(packed_master=P), dict(dtype=4),
])
def test_layer_descriptor(hiplib, kw):
    h = C.c_void_p()
    assert hiplib.wisp_layer_create(C.byref(_desc(**kw)), C.byref(h)) == INVALID
    assert not h.value


def test_work_bytes(hiplib):
    w = hiplib.wisp_moe_mxfp4_work_bytes
    assert w(0, 2, 64, 32, 4) == w(1, 0, 64, 32, 4) == w(1, 2, 64, 32, 0) == 0
    assert w(1 << 26, 64, 64, 32, 4) == 0                # more pairs than 31 bits count
    assert w(1, 2, 64, 32, 4) >= 2 * 32 * 4              # act in float32
    assert w(100, 2, 64, 32, 4) >= 200 * 64 * 4          # y
    # a group of a call fits the call's buffer
    for T in range(13, 64):
        assert w(T, 2, 64, 32, 4) <= w(T + 1, 2, 64, 32, 4)


def test_host_tensors_are_refused():
    u8 = torch.zeros((2, 64, 32), dtype=torch.uint8)
    for call in (lambda: mx.quantize_mxfp4(torch.zeros((2, 64))),
                 lambda: mx.dequantize_mxfp4(u8, u8),
                 lambda: mx.experts_mxfp4(torch.zeros((1, 64), dtype=torch.bfloat16), None, None,
                                          u8, u8, u8, u8),
                 lambda: mx.route_and_experts_mxfp4(torch.zeros((1, 64), dtype=torch.bfloat16),
                                                    None, 2, True, u8, u8, u8, u8)):
        with pytest.raises(ValueError, match="device tensors"):
            call()
