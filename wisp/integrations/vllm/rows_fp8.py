"""Rows of activations before and between the experts' products: the RMS norm
with the residual's addition, and the SwiGLU, with outputs in the rows' own
type or in 8 bits with scales.

The reference leaves both to vLLM; here they make the 8-bit rows that
:func:`wisp.integrations.vllm.grouped_mm.grouped_mm_fp8` reads, so that a row is
rounded once on its way into the product, and a program that sends rows to the
owners of their experts moves half the bytes.

8-bit rows: ``float8_e4m3fn`` codes ``[rows, cols]`` and one float32 scale per
row and group of 128 columns, ``[rows, ceil(cols / 128)]`` (the format of
``wisp_quant_fp8_groups``; here a row's last group may be shorter):
``s = max(max|y|, 1e-10) / 448`` and ``q = y / s`` to the nearest code, from
the float32 ``y``.  A group that holds an infinity or a NaN gets NaN codes.  Rows
of any width are made; the products take those of whole 16 columns.
"""
from __future__ import annotations

import functools

import torch

from wisp_amd import _lib
from wisp_amd._lib import check, lib
from .fused_moe import _require_device

FP8 = torch.float8_e4m3fn
GROUP = 128
_DTYPES = {torch.float32: _lib.WISP_F32, torch.bfloat16: _lib.WISP_BF16}


def _on_device(fn):
    """Runs ``fn`` with its first argument's GPU as the current device, on
    that device's current stream."""
    first = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def call(*args, **kwargs):
        t = args[0] if args else kwargs.get(first)
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"wisp: {fn.__name__} takes device tensors")
        if t.get_device() == torch._C._cuda_getDevice():
            return fn(*args, **kwargs)
        with torch.cuda.device(t.device):
            return fn(*args, **kwargs)
    return call


def _stream(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with contiguous rows (any distance between them)."""
    return t if t.stride()[1] == 1 or t.shape[1] <= 1 else t.contiguous()


def _overlap(t: torch.Tensor, other: torch.Tensor) -> bool:
    """Whether rows of ``t`` and ``other`` (2-D, contiguous rows) share bytes."""
    def of(v):
        size = v.element_size()
        return v.data_ptr(), v.shape[1] * size, (v.stride(0) if v.shape[0] > 1 else 0) * size

    (a, wide_a, step_a), (b, wide_b, step_b) = of(t), of(other)
    if a >= b + (other.shape[0] - 1) * step_b + wide_b or \
            b >= a + (t.shape[0] - 1) * step_a + wide_a:
        return False
    # columns of one buffer: rows interleave without meeting
    return not (step_a == step_b and wide_a <= (b - a) % step_a <= step_a - wide_b) \
        if step_a else True


def _check_apart(name: str, t: torch.Tensor, others) -> None:
    """``t`` is written row by row while the others are read and written: it
    may be one of them, element by element, but not overlap one otherwise."""
    for other, may_be in others:
        if other is None or not t.numel() or not other.numel():
            continue
        other = other if other.dim() == 2 else other[None]
        if may_be and t.data_ptr() == other.data_ptr() and t.dtype == other.dtype and \
                (t.stride(0) == other.stride(0) or t.shape[0] == 1):
            continue
        if _overlap(t, other):
            raise ValueError(f"wisp: {name} overlaps another tensor of the call")


def _check_norm(x, weight, residual, residual_out, out):
    """Raises for what the call does not take."""
    if x.dim() != 2 or weight.dim() != 1 or weight.shape[0] != x.shape[1]:
        raise ValueError("wisp: x is [rows, cols] and weight [cols]")
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"wisp: rows of {x.dtype} (float32 and bfloat16)")
    for t, name in ((weight, "weight"), (residual, "residual")):
        if t is not None and t.dtype != x.dtype and t.dtype != torch.float32:
            raise NotImplementedError("wisp: weight and residual are of x's type or float32")
    for t, name in ((weight, "weight"), (residual, "residual"), (residual_out, "residual_out"),
                    (out, "out")):
        if t is not None:
            _require_device(t, x.device, name)
    if residual is None:
        if residual_out is not None:
            raise ValueError("wisp: residual_out without a residual")
    elif residual.shape != x.shape:
        raise ValueError(f"wisp: residual must be {tuple(x.shape)}")
    rows, cols = x.shape
    if residual_out is not None:
        if residual_out.shape != x.shape or residual_out.dtype != residual.dtype or \
                (cols > 1 and residual_out.stride(1) != 1) or \
                (rows > 1 and residual_out.stride(0) < cols):
            raise ValueError(f"wisp: residual_out must be {tuple(x.shape)} {residual.dtype} "
                             "with contiguous rows")
        _check_apart("residual_out", residual_out, ((x, True), (residual, True), (weight, False)))
    if out is not None:
        if out.shape != x.shape or out.dtype != x.dtype or not out.is_contiguous():
            raise ValueError(f"wisp: out must be a contiguous {tuple(x.shape)} {x.dtype} tensor")
        _check_apart("out", out, ((x, True), (residual, True), (weight, False),
                                  (residual_out, False)))


def _like(x: torch.Tensor) -> torch.Tensor:
    """A new contiguous tensor of ``x``'s shape and type (the quicker way where
    there is one)."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _norm(x, weight, eps, residual, residual_out, out, q, s):
    """The call: checks, then one launch.  (The common call is recognised first:
    the checks take microseconds, as long as a small call's kernel.)"""
    dtype, dev, shape = x.dtype, x.get_device(), x.shape
    if residual_out is not None or out is not None or len(shape) != 2 or dtype not in _DTYPES or \
            weight.dtype != dtype or weight.get_device() != dev or \
            weight.shape != shape[1:] or (residual is not None and (
                residual.dtype != dtype or residual.get_device() != dev or
                residual.shape != shape)):
        _check_norm(x, weight, residual, residual_out, out)
    rows, cols = shape
    if cols > 32768:
        raise NotImplementedError("wisp: norms of more than 32768 columns")
    # (a copy of rows that are not contiguous comes after the check for overlaps)
    x, weight = _rows(x), weight.contiguous()
    codes = scales = to = 0
    if q:
        q = x.new_empty(shape, dtype=FP8)
        s = x.new_empty((rows, -(-cols // GROUP)), dtype=torch.float32)
        codes, scales = q.data_ptr(), s.data_ptr()
    elif out is None:
        out = _like(x)
    if out is not None:
        to = out.data_ptr()
    r = rdt = rs = ro = ros = 0
    if residual is not None:
        residual = _rows(residual)
        if residual_out is None:
            residual_out, ros = _like(residual), cols
        else:
            ros = residual_out.stride(0)
        r, rdt, rs, ro = residual.data_ptr(), _DTYPES[residual.dtype], residual.stride(0), \
            residual_out.data_ptr()
    if rows and cols:
        rc = lib().wisp_add_rms_norm(x.data_ptr(), _DTYPES[dtype], rows, cols, x.stride(0), r, rdt,
                                     rs, ro, ros, weight.data_ptr(), _DTYPES[weight.dtype], eps,
                                     to, codes, scales, _stream(x))
        if rc:
            check(rc, "add_rms_norm")
    return out, q, s, residual_out


@_on_device
def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                 residual: torch.Tensor | None = None, *, out: torch.Tensor | None = None,
                 residual_out: torch.Tensor | None = None):
    """``(out, residual_out)`` of rows ``x [rows, cols]`` (bfloat16 or
    float32): ``r = x + residual`` rounded once to the residual's type (``x``
    itself and ``None`` without a residual), ``out = r / sqrt(mean(r**2) +
    eps) * weight`` in float32, rounded once to ``x``'s type.  The weight and
    the residual are of ``x``'s type or float32.  Rows may lie any distance
    apart; up to 32768 columns.  ``out`` may be ``x`` or ``residual``, and
    ``residual_out`` may be ``residual`` or ``x``, but not one the other."""
    out, _, _, residual_out = _norm(x, weight, eps, residual, residual_out, out, False, None)
    return out, residual_out


@_on_device
def add_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                     residual: torch.Tensor | None = None, *, out: torch.Tensor | None = None,
                     residual_out: torch.Tensor | None = None):
    """:func:`add_rms_norm` in 8 bits: ``(codes, scales, residual_out)``.  With
    ``out`` the normalised rows also go there in ``x``'s type (for a router
    that reads them), from the same float32 values."""
    _, q, s, residual_out = _norm(x, weight, eps, residual, residual_out, out, True, None)
    return q, s, residual_out


@_on_device
def silu_mul_fp8(h: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """SwiGLU of a product's rows ``h [rows, 2 * I]`` (gate, then up; bfloat16
    or float32, rows any distance apart) in 8 bits: codes ``[rows, I]`` and
    scales ``[rows, ceil(I / 128)]`` of ``silu(h[:, :I]) * h[:, I:]``."""
    if h.dim() != 2 or h.shape[1] % 2:
        raise ValueError("wisp: h is [rows, 2 * I]")
    if h.dtype not in _DTYPES:
        raise NotImplementedError(f"wisp: rows of {h.dtype} (float32 and bfloat16)")
    if h.shape[1] >= 1 << 31:
        raise NotImplementedError("wisp: rows of 2^31 columns")
    h = _rows(h)
    rows, inter = h.shape[0], h.shape[1] // 2
    q = h.new_empty((rows, inter), dtype=FP8)
    s = h.new_empty((rows, -(-inter // GROUP)), dtype=torch.float32)
    if rows and inter:
        rc = lib().wisp_silu_mul_fp8(h.data_ptr(), _DTYPES[h.dtype], rows, inter, h.stride(0),
                                     q.data_ptr(), s.data_ptr(), _stream(h))
        if rc:
            check(rc, "silu_mul_fp8")
    return q, s


__all__ = ["add_rms_norm", "add_rms_norm_fp8", "silu_mul_fp8"]
