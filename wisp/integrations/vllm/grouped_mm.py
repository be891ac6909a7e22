"""Matrix products grouped by expert, over rows that are sorted by expert.

An expert-parallel rank gets its tokens' rows from an all-to-all in the order of
its experts, as many of each as the routing made, in a buffer that may hold
more.  The reference runs whole experts over (token, expert) pairs of one GPU
only; these products are the parts of such a rank's experts::

    q, s, residual = add_rms_norm_fp8(x, weight, eps, residual)
    ...                                            # rows to the owners of their experts
    h = grouped_mm_fp8(q, s, w13, s13, ends)       # [rows, 2 * I]
    a, sa = silu_mul_fp8(h)
    y = grouped_mm_fp8(a, sa, w2, s2, ends)        # [rows, H]

``ends [E]`` (int32, on the device, never read by the host): group ``e`` is the
rows ``[ends[e - 1], ends[e])``, from 0 for the first.  An end outside ``[0,
rows]`` counts as 0 or ``rows``, one below an earlier end as that one, so groups
never overlap.  Rows behind the last group are left as they are in a given
``out`` and are zero in a new one.  Up to 512 experts of fewer than 2^21 outputs;
weights are ``[E, N, K]`` (``w13``, ``w2`` as the MoE layers hold them), each row
contiguous, an expert's less than 2 GiB and its rows less than 16 MiB apart (rows of
``x``, and of its scales, less than 4 MiB).

The kernel goes by the sizes that the host knows: experts, outputs, columns and
the rows of the buffer, however few of them ``ends`` puts into groups.  A buffer
much larger than its rows takes the kernel of a full one: where a program can,
it passes as many rows as it may have.  The order of a row's sum goes by the
kernel and by its expert's number in the call, so the same call gives the same
bytes again, but a token's row may have other last bits (each within the bound
of a float32 sum) in another batch or on a rank that numbers its experts
otherwise.
"""
from __future__ import annotations

import torch

from wisp_amd import _lib
from wisp_amd._lib import check, lib
from .fused_moe import _require_device
from .rows_fp8 import FP8, GROUP, _DTYPES, _check_apart, _on_device, _stream


def _sizes(x, w, ends) -> tuple[int, int, int, int, int, int]:
    """``(M, E, N, K)`` of rows, weights and ends, and the elements from expert to
    expert and from row to row of the weights (a single one's stride may be
    anything)."""
    try:
        (M, C), (E, N, K), (groups,) = x.shape, w.shape, ends.shape
    except ValueError:
        raise ValueError("wisp: grouped products take rows [M, K], weights [E, N, K] and "
                         "ends [E]") from None
    if K != C or groups != E or not E:
        raise ValueError("wisp: grouped products take rows [M, K], weights [E, N, K] and ends "
                         f"[E], got {(M, C)}, {(E, N, K)}, {(groups,)}")
    if ends.dtype != torch.int32:
        raise ValueError("wisp: ends are int32")
    dev = x.get_device()
    if w.get_device() != dev or ends.get_device() != dev:
        _require_device(w, x.device, "w")
        _require_device(ends, x.device, "ends")
    step, ld, one = w.stride()
    if K > 1 and one != 1:
        raise ValueError("wisp: each row of w must be contiguous")
    if M >= 1 << 31 or N >= 1 << 21 or K >= 1 << 31:
        raise NotImplementedError("wisp: grouped products take fewer than 2^31 rows and columns "
                                  "and 2^21 outputs")
    return M, E, N, K, step if E > 1 else 0, ld if N > 1 else K


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First and one past the last byte that ``t`` may touch."""
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * \
        t.element_size()


def _aligned_rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` with contiguous rows that start 16-byte aligned."""
    step, one = x.stride()
    if one == 1 and step >= x.shape[1] and (x.data_ptr() | step * x.element_size()) % 16 == 0:
        return x
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def _output(x, N, dtype, out, inputs, weights) -> torch.Tensor:
    if out is None:
        return x.new_empty((x.shape[0], N), dtype=dtype)
    if out.shape != (x.shape[0], N) or out.dtype != dtype or not out.is_contiguous():
        raise ValueError(f"wisp: out must be a contiguous {(x.shape[0], N)} {dtype} tensor")
    if out.get_device() != x.get_device():
        _require_device(out, x.device, "out")
    _check_apart("out", out, [(t, False) for t in inputs])
    if out.numel():
        first, last = _span(out)
        for t in weights:  # (also the room between their experts)
            a, b = _span(t)
            if t.numel() and a < last and first < b:
                raise ValueError("wisp: out overlaps another tensor of the call")
    return out


@_on_device
def grouped_mm(x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor, *,
               dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[i] = w[e] @ x[i]`` for the rows ``i`` of group ``e``: bfloat16
    ``x [M, K]`` and ``w [E, N, K]``, float32 sums, rounded once to ``dtype``
    (bfloat16 or float32; a given ``out`` is of that type).  K is a multiple of
    8; rows of ``x`` may lie any distance apart, experts and rows of ``w`` any
    multiple of 16 bytes, and ``w`` starts at one.  A given ``out`` may start
    anywhere (a bfloat16 one between two dwords is stored value by value,
    which takes longer)."""
    M, E, N, K, step, w_ld = _sizes(x, w, ends)
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16:
        raise NotImplementedError("wisp: grouped_mm takes bfloat16 rows and weights")
    if dtype not in _DTYPES:
        raise NotImplementedError(f"wisp: grouped_mm cannot give {dtype} (float32 and bfloat16)")
    x, ends = _aligned_rows(x), ends.contiguous()
    given = out is not None
    out = _output(x, N, dtype, out, (x, ends), (w,))
    if M and N:
        rc = lib().wisp_grouped_mm(x.data_ptr(), x.stride(0) if M > 1 else K, w.data_ptr(),
                                   step, w_ld, ends.data_ptr(), E, M, N, K, out.data_ptr(),
                                   _DTYPES[dtype], not given, _stream(x))
        if rc:
            check(rc, "grouped_mm")
    return out


@_on_device
def grouped_mm_fp8(q: torch.Tensor, s: torch.Tensor, w: torch.Tensor, ws: torch.Tensor,
                   ends: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`grouped_mm` over block FP8, in bfloat16: codes ``q [M, K]`` with
    scales ``s [M, ceil(K / 128)]`` (``add_rms_norm_fp8``, ``silu_mul_fp8``)
    and codes ``w [E, N, K]`` with block scales ``ws [E, ceil(N / 128),
    ceil(K / 128)]``, all codes ``float8_e4m3fn`` and scales float32.  K is a
    multiple of 16.  The products of 128 columns are summed by the matrix
    instruction, scaled and summed in float32, and rounded once.  The
    instruction's sums are right to some 2^-16 of the products' sizes on
    ordinary quantised rows, to 2^-12 on codes of the full range: there is no
    float32 output."""
    M, E, N, K, step, w_ld = _sizes(q, w, ends)
    if q.dtype != FP8 or w.dtype != FP8:
        raise NotImplementedError("wisp: grouped_mm_fp8 takes float8_e4m3fn codes")
    G, B = -(-K // GROUP), -(-N // GROUP)
    if s.shape != (M, G) or ws.shape != (E, B, G) or s.dtype != torch.float32 or \
            ws.dtype != torch.float32:
        raise ValueError(f"wisp: scales are float32, s {(M, G)} and ws {(E, B, G)}")
    if s.get_device() != q.get_device() or ws.get_device() != q.get_device():
        _require_device(s, q.device, "s")
        _require_device(ws, q.device, "ws")
    if not ws.is_contiguous() and not ws[0].is_contiguous():
        raise ValueError("wisp: each expert's block scales must be contiguous")
    q, ends = _aligned_rows(q), ends.contiguous()
    if (s.stride(1) != 1 and G > 1) or s.stride(0) < G:
        s = s.contiguous()
    given = out is not None
    out = _output(q, N, torch.bfloat16, out, (q, s, ends), (w, ws))
    if M and N:
        rc = lib().wisp_grouped_mm_fp8(
            q.data_ptr(), q.stride(0) if M > 1 else K, s.data_ptr(), s.stride(0) if M > 1 else G,
            w.data_ptr(), step, w_ld, ws.data_ptr(), ws.stride(0) if E > 1 else 0,
            ends.data_ptr(), E, M, N, K,
            out.data_ptr(), not given, _stream(q))
        if rc:
            check(rc, "grouped_mm_fp8")
    return out


__all__ = ["grouped_mm", "grouped_mm_fp8"]
