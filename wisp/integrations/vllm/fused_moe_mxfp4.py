"""MXFP4 experts for MI355X: quantising weights to 4-bit microscaled floating
point, reading them back, and the MoE layer over such weights.

The reference pages bf16 and block-FP8 experts only; this format has no
counterpart there.  An expert in MXFP4 is 17/32 of a byte a weight: 3.76 times
fewer bytes over the host link and from HBM than in bf16, 1.88 times fewer
than in FP8.

Format.  A row's values in blocks of 32; each value a 4-bit E2M1 code (two to a
byte, the earlier value in the low half), each block one E8M0 scale byte ``s``;
a value is ``E2M1(code) * 2**(s - 127)``, ``s == 255`` is NaN.  Weights are
``uint8`` tensors: codes ``w13 [E, 2I, H/2]``, ``w2 [E, H, I/2]``, scales
``s13 [E, 2I, H/32]``, ``s2 [E, H, I/32]``.  Activations are bfloat16, products
are summed in float32 and the output is rounded to bfloat16 once.  The SwiGLU
result stays in float32 in calls of few tokens (at most 12, by the whole call's
tokens, shape and number of experts) and is rounded to bfloat16 once in all
others, so a token's bytes may differ between a small and a larger call.

``WispMoEStateMxfp4`` is the paging state over such experts: masters in pinned
host memory, one ``[w13 | w2 | s13 | s2]`` slab per expert, the same pager,
page-in, prefetch and resize as the bf16 state's.  ``WISP_EXPERT_FORMAT=mxfp4``
makes ``install_wisp_moe`` quantise a bf16 layer's experts when its weights are
loaded and run the layer on such a state.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from wisp_amd import _lib
from wisp_amd._lib import check, lib
from .fused_moe import (WispMoEState, _check_out, _Mode, _require_device, _resolve_pagein_engine,
                        _resolve_pagein_streams, _Workspace)

BLOCK = 32
_DTYPES = {torch.float32: _lib.WISP_F32, torch.bfloat16: _lib.WISP_BF16}


def _on_device(fn):
    """Runs ``fn`` with its first argument's GPU as the current device, on
    that device's current stream."""
    first = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def call(*args, **kwargs):
        t = args[0] if args else kwargs.get(first)
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"wisp.mxfp4: {fn.__name__} takes device tensors")
        if t.get_device() == torch._C._cuda_getDevice():  # (current_device() without its checks)
            return fn(*args, **kwargs)
        with torch.cuda.device(t.device):
            return fn(*args, **kwargs)
    return call


def _stream(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.get_device())


@_on_device
def quantize_mxfp4(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``w [..., C]`` (float32 or bfloat16, C a multiple of 32) -> codes
    ``[..., C/2]`` and scales ``[..., C/32]``.  A block's scale is
    ``2**(floor(log2(max|w|)) - 2)``, no smaller than ``2**-127``; values are
    rounded to the nearest code (ties to the even one) and saturate at 6 times
    the scale.  A block with an infinity or a NaN reads back as NaNs."""
    if w.dtype not in _DTYPES:
        raise NotImplementedError(f"wisp.mxfp4: cannot quantise {w.dtype} (float32 and bfloat16)")
    if w.dim() < 1 or w.shape[-1] % BLOCK:
        raise ValueError("wisp.mxfp4: the last dimension must be a multiple of 32")
    w = w.contiguous()
    if w.data_ptr() % 16:
        w = w.clone()
    C = w.shape[-1]
    codes = torch.empty((*w.shape[:-1], C // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((*w.shape[:-1], C // BLOCK), dtype=torch.uint8, device=w.device)
    if w.numel():
        # (one run of blocks whatever the shape: a row's length may exceed the call's int)
        check(lib().wisp_quant_mxfp4(w.data_ptr(), _DTYPES[w.dtype], w.numel() // BLOCK, BLOCK,
                                     codes.data_ptr(), scales.data_ptr(), _stream(w)),
              "quantize_mxfp4")
    return codes, scales


@_on_device
def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor,
                     dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of codes ``[..., C/2]`` and scales ``[..., C/32]`` as
    ``[..., C]`` in ``dtype`` (bfloat16 or float32; both hold them exactly, but
    for magnitudes of ``2**128`` or more, which become infinities)."""
    if dtype not in _DTYPES:
        raise NotImplementedError(f"wisp.mxfp4: cannot read back as {dtype} "
                                  "(float32 and bfloat16)")
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError("wisp.mxfp4: codes and scales are uint8")
    if codes.dim() < 1 or scales.shape != (*codes.shape[:-1], codes.shape[-1] // 16) or \
            codes.shape[-1] % 16:
        raise ValueError(f"wisp.mxfp4: codes {tuple(codes.shape)} and scales "
                         f"{tuple(scales.shape)} disagree (16 bytes of codes a scale)")
    if scales.get_device() != codes.get_device():
        _require_device(scales, codes.device, "scales")
    codes, scales = codes.contiguous(), scales.contiguous()
    if codes.data_ptr() % 4:
        codes = codes.clone()
    C = 2 * codes.shape[-1]
    out = torch.empty((*codes.shape[:-1], C), dtype=dtype, device=codes.device)
    if out.numel():
        check(lib().wisp_dequant_mxfp4(codes.data_ptr(), scales.data_ptr(),  # (as above)
                                       out.numel() // BLOCK, BLOCK, out.data_ptr(),
                                       _DTYPES[dtype], _stream(codes)),
              "dequantize_mxfp4")
    return out


def _check_weights(x, w13, w2, s13, s2) -> tuple[int, int, int]:
    """``(E, H, I)`` of MXFP4 expert tensors beside activations ``x [T, H]``."""
    if x.dtype != torch.bfloat16:
        raise NotImplementedError("wisp.mxfp4: activations must be bfloat16")
    if x.dim() != 2 or w13.dim() != 3 or w2.dim() != 3:
        raise ValueError("wisp.mxfp4: x is [T, H], w13 [E, 2I, H/2], w2 [E, H, I/2]")
    H = x.shape[1]
    E, I = w13.shape[0], 2 * w2.shape[2]
    if w13.shape != (E, 2 * I, H // 2) or w2.shape != (E, H, I // 2) or \
            s13.shape != (E, 2 * I, H // BLOCK) or s2.shape != (E, H, I // BLOCK):
        raise ValueError(f"wisp.mxfp4: for x [T, {H}], E = {E} and I = {I}, w13 is "
                         f"{(E, 2 * I, H // 2)}, w2 {(E, H, I // 2)}, s13 "
                         f"{(E, 2 * I, H // BLOCK)} and s2 {(E, H, I // BLOCK)}")
    dev = x.get_device()
    for t in (w13, w2, s13, s2):
        if t.dtype != torch.uint8:
            raise ValueError("wisp.mxfp4: codes and scales are uint8 tensors")
        if t.get_device() != dev:
            _require_device(t, x.device, "an expert tensor")
        if not t.is_contiguous() and (t.stride(2) != 1 or t.stride(1) != t.shape[2]):
            raise ValueError("wisp.mxfp4: each expert of w13, w2, s13 and s2 must be contiguous")
    return E, H, I


@functools.lru_cache(maxsize=256)
def _layout(T: int, K: int, H: int, I: int, nslots: int) -> tuple[int, int, int]:
    """Byte offset of a call's routing and work buffer behind its act, and the
    work buffer's size."""
    routing = -(-T * K * I * 2 // 256) * 256
    work = routing + -(-T * K * 8 // 256) * 256
    return routing, work, lib().wisp_moe_mxfp4_work_bytes(T, K, H, I, nslots)


def _output(x, out):
    if out is None:
        return torch.empty_like(x)
    _check_out(out, x)
    return out


@_on_device
def experts_mxfp4(x: torch.Tensor, topk_w: torch.Tensor, slots: torch.Tensor, w13: torch.Tensor,
                  w2: torch.Tensor, s13: torch.Tensor, s2: torch.Tensor,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """SwiGLU experts over MXFP4 weights with the routing-order combine:
    ``out[t] = sum_k topk_w[t, k] * expert(slots[t, k], x[t])``.  ``x [T, H]``
    bfloat16, ``topk_w [T, K]`` float32, ``slots [T, K]`` int32; a slot outside
    ``[0, E)`` (say -1) contributes nothing."""
    E, H, I = _check_weights(x, w13, w2, s13, s2)
    T = x.shape[0]
    if slots.dim() != 2 or slots.shape[0] != T or topk_w.shape != slots.shape or \
            slots.dtype != torch.int32 or topk_w.dtype != torch.float32:
        raise ValueError(f"wisp.mxfp4: topk_w float32 and slots int32 must be [{T}, K]")
    for t in (slots, topk_w):
        if t.get_device() != x.get_device():
            _require_device(t, x.device, "the routing")
    K = slots.shape[1]
    x, slots, topk_w = x.contiguous(), slots.contiguous(), topk_w.contiguous()
    out = _output(x, out)
    if T == 0:
        return out
    # one allocation of the call's own, so that calls on other streams, or
    # captured into other graphs, share nothing
    _, work, nbytes = _layout(T, K, H, I, E)
    buf = torch.empty(work + nbytes, dtype=torch.uint8, device=x.device)
    p = buf.data_ptr()
    check(lib().wisp_moe_experts_mxfp4(
        x.data_ptr(), T, H, I, K, topk_w.data_ptr(), slots.data_ptr(), E, w13.data_ptr(),
        w13.stride(0), s13.data_ptr(), s13.stride(0), w2.data_ptr(), w2.stride(0), s2.data_ptr(),
        s2.stride(0), p, out.data_ptr(), p + work, nbytes, _stream(x)), "experts_mxfp4")
    return out


@_on_device
def route_and_experts_mxfp4(x: torch.Tensor, router_logits: torch.Tensor, top_k: int,
                            renormalize: bool, w13: torch.Tensor, w2: torch.Tensor,
                            s13: torch.Tensor, s2: torch.Tensor,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """The whole MoE layer, all MXFP4 experts resident in device tensors:
    softmax routing of ``router_logits [T, E]`` (top-k by logit, ties to the
    lower id), then :func:`experts_mxfp4` with slot = expert id."""
    E, H, I = _check_weights(x, w13, w2, s13, s2)
    T, K = x.shape[0], int(top_k)
    if router_logits.shape != (T, E):
        raise ValueError(f"wisp.mxfp4: router_logits must be [{T}, {E}]")
    if not 1 <= K <= E:
        raise ValueError(f"wisp.mxfp4: top_k={top_k} outside [1, {E}]")
    if router_logits.get_device() != x.get_device():
        _require_device(router_logits, x.device, "router_logits")
    if router_logits.dtype not in _DTYPES:
        router_logits = router_logits.float()
    x, router_logits = x.contiguous(), router_logits.contiguous()
    out = _output(x, out)
    if T == 0:
        return out
    routing, work, nbytes = _layout(T, K, H, I, E)
    buf = torch.empty(work + nbytes, dtype=torch.uint8, device=x.device)  # as above
    p = buf.data_ptr()
    check(lib().wisp_moe_layer_mxfp4(
        x.data_ptr(), router_logits.data_ptr(), _DTYPES[router_logits.dtype], T, H, I, E, K,
        int(bool(renormalize)), p + routing, p + routing + 4 * T * K,
        w13.data_ptr(), w13.stride(0), s13.data_ptr(), s13.stride(0), w2.data_ptr(), w2.stride(0),
        s2.data_ptr(), s2.stride(0), p, out.data_ptr(), p + work, nbytes, _stream(x)),
        "route_and_experts_mxfp4")
    return out


# ---------------------------------------------------------------------------
# The paging state
# ---------------------------------------------------------------------------


class Mxfp4SlabLayout:
    """Byte layout of one expert's ``[w13 | w2 | s13 | s2]`` slab."""

    def __init__(self, hidden: int, inter: int) -> None:
        H, I = int(hidden), int(inter)
        if H < BLOCK or I < BLOCK or H % BLOCK or I % BLOCK:
            raise ValueError(f"wisp.mxfp4: hidden={H} and inter={I} must be multiples of {BLOCK}")
        self.hidden, self.inter = H, I
        self.parts = ((2 * I, H // 2), (H, I // 2), (2 * I, H // BLOCK), (H, I // BLOCK))
        self.offsets, end = [], 0
        for rows, cols in self.parts:
            self.offsets.append(end)
            end += rows * cols
        self.used = end
        self.slab = -(-end // 256) * 256

    def views(self, buf: torch.Tensor):
        """``buf [N, slab] uint8`` -> ``(w13, w2, s13, s2)`` views of N experts."""
        base = buf.storage_offset()
        return tuple(torch.as_strided(buf, (buf.shape[0], rows, cols), (self.slab, cols, 1),
                                      base + off)
                     for (rows, cols), off in zip(self.parts, self.offsets))


def mxfp4_slab_masters(num_experts: int, hidden: int, inter: int, pin: bool = True):
    """Host masters as one slab per expert: ``(buf, w13, w2, s13, s2)``, zero
    codes with scale 1."""
    lay = Mxfp4SlabLayout(hidden, inter)
    buf = torch.zeros((num_experts, lay.slab), dtype=torch.uint8, pin_memory=pin)
    w13, w2, s13, s2 = lay.views(buf)
    s13.fill_(127)
    s2.fill_(127)
    return buf, w13, w2, s13, s2


def quantize_masters_mxfp4(w13: torch.Tensor, w2: torch.Tensor, device) -> tuple:
    """``w13 [E, 2I, H]`` and ``w2 [E, H, I]`` (bfloat16 or float32, host or
    device memory) -> pinned host masters ``(w13, w2, s13, s2)`` in MXFP4, one
    slab per expert, quantised on ``device`` an expert at a time."""
    if w13.dim() != 3 or w2.dim() != 3 or w13.shape[0] != w2.shape[0] or \
            w13.shape[1] != 2 * w2.shape[2] or w13.shape[2] != w2.shape[1]:
        raise ValueError("wisp.mxfp4: experts are w13 [E, 2I, H] and w2 [E, H, I]")
    E, H, I = w13.shape[0], w13.shape[2], w2.shape[2]
    _, *views = mxfp4_slab_masters(E, H, I)
    for e in range(E):
        (q13, s13), (q2, s2) = (quantize_mxfp4(w[e].to(device)) for w in (w13, w2))
        for dst, src in zip(views, (q13, q2, s13, s2)):
            dst[e].copy_(src)
    return tuple(views)


class WispMoEStateMxfp4(WispMoEState):
    """Per-layer paging state over MXFP4 experts.

    ``cpu_w13 [E, 2I, H/2]``, ``cpu_w2 [E, H, I/2]`` codes and ``cpu_s13``,
    ``cpu_s2`` scales, ``uint8`` host tensors; pinned ones (views of one slab
    per expert, as :func:`quantize_masters_mxfp4` makes them) page in by the copy
    kernel, an expert a copy.  Routing, the pager, prefetch and resize are the
    unquantised state's; activations and outputs are bfloat16.
    """

    def __init__(self, cpu_w13: torch.Tensor, cpu_w2: torch.Tensor, cpu_s13: torch.Tensor,
                 cpu_s2: torch.Tensor, cap_experts: int, mode: str, device,
                 layer_idx: int) -> None:
        if cpu_w13.dim() != 3 or cpu_w2.dim() != 3:
            raise ValueError("wisp.mxfp4: cpu_w13 is [E, 2I, H/2], cpu_w2 [E, H, I/2]")
        E, H, I = cpu_w13.shape[0], 2 * cpu_w13.shape[2], 2 * cpu_w2.shape[2]
        lay = Mxfp4SlabLayout(H, I)
        masters = (cpu_w13, cpu_w2, cpu_s13, cpu_s2)
        for t, name, part in zip(masters, ("cpu_w13", "cpu_w2", "cpu_s13", "cpu_s2"), lay.parts):
            if t.device.type != "cpu":
                raise ValueError(f"wisp.mxfp4: {name} must live in host memory")
            if t.dtype != torch.uint8 or t.shape != (E, *part):
                raise ValueError(f"wisp.mxfp4: {name} must be a uint8 {(E, *part)} tensor")
            if t.stride(2) != 1 or t.stride(1) != part[1]:
                raise ValueError(f"wisp.mxfp4: each expert of {name} must be contiguous")
        if not 1 <= cap_experts <= E:
            raise ValueError(f"cap_experts={cap_experts} outside [1, {E}]")
        self._layout = lay
        self.layer_idx = int(layer_idx)
        self.num_experts, self.cap_experts = int(E), int(cap_experts)
        self.mode = mode
        self.hidden, self.inter = lay.hidden, lay.inter
        self.dtype = torch.bfloat16  # activations
        self.cpu_w13, self.cpu_w2, self.cpu_s13, self.cpu_s2 = masters
        self.device = torch.device(device)
        self._alloc_scratch(self.cap_experts)
        dev = self.device
        self.expert_map_device = torch.full((E,), -1, dtype=torch.int32, device=dev)
        self._counters = torch.zeros(8, dtype=torch.int64, device=dev)
        self.stats_pred_hits = 0
        self._pf_record = None
        self._pf_words = 0
        self._pf_n = 0
        self._ws = _Workspace(dev, self.hidden, self.inter, torch.bfloat16, mxfp4_experts=int(E))
        self._last_pairs = 0
        self._handle = C.c_void_p()
        self._desc = self._make_desc()
        check(lib().wisp_layer_create(C.byref(self._desc), C.byref(self._handle)),
              "wisp_layer_create")

    @property
    def slot_bytes(self) -> int:
        return self._layout.used

    @property
    def packed_bytes_per_expert(self) -> int:
        return self._layout.used

    def _alloc_scratch(self, cap: int) -> None:
        lay = self._layout
        self._scratch = torch.empty((cap, lay.slab), dtype=torch.uint8, device=self.device)
        self.scratch_w13, self.scratch_w2, self.scratch_s13, self.scratch_s2 = \
            lay.views(self._scratch)
        self._slot_to_expert = torch.full((cap,), -1, dtype=torch.int32, device=self.device)
        self._lru_tick = torch.zeros(cap, dtype=torch.int64, device=self.device)

    def _make_desc(self) -> "_lib.LayerDesc":
        lay = self._layout
        d = _lib.LayerDesc()
        d.struct_bytes = C.sizeof(_lib.LayerDesc)
        d.num_experts, d.cap = self.num_experts, self.cap_experts
        d.hidden, d.inter = self.hidden, self.inter
        d.dtype = _lib.WISP_MXFP4
        d.mode = _lib.WISP_MODE_RESIDENT if self.mode == _Mode.RESIDENT else _lib.WISP_MODE_PAGED
        d.pagein_streams = _resolve_pagein_streams()
        d.pagein_engine = _resolve_pagein_engine()
        sizes = [rows * cols for rows, cols in lay.parts]
        d.w13_elems, d.w2_elems, d.s13_elems, d.s2_elems = sizes
        for part in ("w13", "w2", "s13", "s2"):
            scratch, master = getattr(self, "scratch_" + part), getattr(self, "cpu_" + part)
            setattr(d, "scratch_" + part, scratch.data_ptr())
            setattr(d, f"scratch_{part}_stride", lay.slab)
            setattr(d, "master_" + part, master.data_ptr())
            setattr(d, f"master_{part}_stride", master.stride(0))
        d.expert_map = self.expert_map_device.data_ptr()
        d.slot_to_expert = self._slot_to_expert.data_ptr()
        d.lru_tick = self._lru_tick.data_ptr()
        d.counters = self._counters.data_ptr()
        return d


__all__ = ["quantize_mxfp4", "dequantize_mxfp4", "experts_mxfp4", "route_and_experts_mxfp4",
           "Mxfp4SlabLayout", "mxfp4_slab_masters", "quantize_masters_mxfp4", "WispMoEStateMxfp4"]
