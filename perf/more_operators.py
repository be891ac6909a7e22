"""Performance cases of the operators around and inside the experts of a rank
that receives its tokens' rows sorted by expert: the RMS norm with the
residual's addition, with its output in bfloat16 / float32 or in 8 bits with
scales; matrix products grouped by expert with ragged sizes, in bfloat16 and in
block FP8; and the SwiGLU between two such products, with its output in 8 bits.

8-bit rows: float8_e4m3fn codes with one float32 scale per row and group of 128
columns (the last group of a row may be shorter); weights in block FP8 have one
float32 scale per block of 128 x 128.  Group e of a grouped product is the rows
[ends[e - 1], ends[e]) of x; rows behind the last group come out as zeros.

With ``own`` false, ``run`` computes the operators from elementary torch
operations in float32, rounded once at the end; with ``own`` true it calls
``wisp.integrations.vllm.rows_fp8`` and ``wisp.integrations.vllm.grouped_mm``.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
GROUP = 128
TOP = 448.0
LEAST = 1e-10
WEIGHT_STD = 0.02
FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

# hidden, inter, experts, top_k
LAYERS = {
    "toy": (512, 256, 16, 2),
    "odd": (1056, 352, 24, 3),
    "qwen3": (2048, 768, 128, 8),
    "mixtral": (4096, 14336, 8, 2),
}


def _norm(name, op, rows, cols, dtype="bf16", residual=True):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "dtype": dtype,
            "residual": residual}


def _silu(name, rows, inter):
    return {"name": name, "op": "silu8", "rows": rows, "inter": inter}


def _grouped(name, op, layer, product, tokens, ranks=1, skew=0.0, dtype="bf16"):
    return {"name": name, "op": op, "layer": layer, "product": product, "tokens": tokens,
            "ranks": ranks, "skew": skew, "dtype": dtype}


def listed():
    return [
        # bs=1 generation: the norm in front of a bf16 layer.
        _norm("norm-decode-1", "norm", 1, 2048),
        # In front of FP8 experts: odd sizes in float32, the first norm of a
        # model (no residual yet); a large prompt chunk.
        _norm("norm8-odd-f32", "norm8", 333, 1375, "f32", False),
        _norm("norm8-prompt-8192", "norm8", 8192, 4096),
        # The SwiGLU between the products: odd sizes, a large chunk.
        _silu("silu8-odd-231", 231, 352),
        _silu("silu8-qwen3-65536", 65536, 768),
        # bs=1 generation: eight experts of one row each.
        _grouped("mm-qwen3-w13-1", "mm", "qwen3", "w13", 1),
        # A rank's share (16 of 128 experts) of an odd number of tokens, some
        # experts liked more, in a buffer with room to spare.
        _grouped("mm-qwen3-w2-rank-777", "mm", "qwen3", "w2", 777, 8, 0.5),
        # A large prompt chunk in bfloat16.
        _grouped("mm-qwen3-w13-8192", "mm", "qwen3", "w13", 8192),
        # Odd sizes with a float32 output, as a caller that sums many experts'
        # outputs itself takes it.
        _grouped("mm-odd-w2-77-f32", "mm", "odd", "w2", 77, 1, 0.5, "f32"),
        # In FP8 (bf16 out): batched generation, odd sizes, a chunk through few
        # large experts.
        _grouped("mm8-qwen3-w13-32", "mm8", "qwen3", "w13", 32),
        _grouped("mm8-odd-w13-77", "mm8", "odd", "w13", 77, 1, 0.5),
        _grouped("mm8-mixtral-w13-2000", "mm8", "mixtral", "w13", 2000),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: rows of other sizes, the same layers
    at other token counts, either product, whole or a rank's share."""
    op = rng.choice(["norm", "norm8", "silu8", "mm", "mm", "mm8", "mm8"])
    if op in ("norm", "norm8"):
        cols = 8 * _log_int(rng, 8, 1024) if rng.random() < 0.7 else _log_int(rng, 64, 8192)
        c = _norm("", op, _log_int(rng, 1, 8192 * 4096 // max(cols, 4096)), cols,
                  rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.7)
    elif op == "silu8":
        inter = 8 * _log_int(rng, 8, 1792)
        c = _silu("", _log_int(rng, 1, 65536 * 768 // max(inter, 768)), inter)
    else:
        layer = rng.choice(["toy", "odd", "qwen3", "qwen3", "mixtral"])
        most = {"toy": 8192, "odd": 8192, "qwen3": 8192, "mixtral": 800}[layer]
        ranks = rng.choice([1, 1, 2, 8]) if layer != "mixtral" else rng.choice([1, 2])
        c = _grouped("", op, layer, rng.choice(["w13", "w2"]), _log_int(rng, 1, most), ranks,
                     round(rng.choice([0.0, rng.uniform(0.0, 0.7)]), 2),
                     rng.choice(["bf16", "bf16", "f32"]) if op == "mm" else "bf16")
    del c["name"]
    return c


def _sizes(case):
    """Local experts, output columns, input columns and rows of the buffer: all
    pairs of the tokens, or a rank's share of them and a quarter more."""
    H, I, E, K = LAYERS[case["layer"]]
    N, C = (2 * I, H) if case["product"] == "w13" else (H, I)
    pairs = case["tokens"] * K
    rows = pairs if case["ranks"] == 1 else -(-pairs * 5 // (4 * case["ranks"]))
    return E // case["ranks"], N, C, rows


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _generator(seed, which):
    return torch.Generator(device="cuda").manual_seed(8 * seed + which)


def _quantize_rows(v):
    """Codes and scales of the float32 rows ``v [M, C]``."""
    M, C = v.shape
    G = -(-C // GROUP)
    g = torch.nn.functional.pad(v, (0, G * GROUP - C)).view(M, G, GROUP)
    s = g.abs().amax(dim=2).clamp(min=LEAST) / TOP
    q = (g / s[..., None]).clamp(-TOP, TOP).view(M, G * GROUP)[:, :C]
    return q.to(FP8), s


def _spread(ws, N, C):
    """Block scales ``[..., N/128, C/128]`` over the weights ``[..., N, C]``."""
    return ws.repeat_interleave(GROUP, dim=-2)[..., :N, :].repeat_interleave(
        GROUP, dim=-1)[..., :C]


def _quantize_blocks(w):
    """Codes and block scales of one weight ``w [N, C]``."""
    N, C = w.shape
    n, c = -(-N // GROUP), -(-C // GROUP)
    b = torch.nn.functional.pad(w, (0, c * GROUP - C, 0, n * GROUP - N))
    ws = b.view(n, GROUP, c, GROUP).abs().amax(dim=(1, 3)).clamp(min=LEAST) / TOP
    return (w / _spread(ws, N, C)).clamp(-TOP, TOP).to(FP8), ws


def _norm_inputs(case, seed):
    """The block's output, the residual stream beside it (of larger values, as
    it grows through a model) and the norm's weight, near one."""
    g = _generator(seed, 0)
    shape, dtype = (case["rows"], case["cols"]), DTYPES[case["dtype"]]
    x = torch.randn(shape, generator=g, device="cuda").to(dtype)
    w = (1.0 + 0.1 * torch.randn(case["cols"], generator=g, device="cuda")).to(dtype)
    r = None
    if case["residual"]:
        r = (3.0 * torch.randn(shape, generator=g, device="cuda")).to(dtype)
    return x, r, w


def _silu_inputs(case, seed):
    return torch.randn((case["rows"], 2 * case["inter"]), generator=_generator(seed, 1),
                       device="cuda").to(torch.bfloat16)


def _ends(case, seed):
    """Ends of the local experts' rows: every token's top_k of all experts, some
    of them more liked than others where ``skew`` is not 0."""
    _, _, E, K = LAYERS[case["layer"]]
    g = _generator(seed, 2)
    score = torch.randn((case["tokens"], E), generator=g, device="cuda")
    score += case["skew"] * torch.randn(E, generator=g, device="cuda")
    ids = score.topk(K, dim=1).indices.reshape(-1)
    local, _, _, rows = _sizes(case)
    n = torch.zeros(E, dtype=torch.int64, device="cuda").index_add_(
        0, ids, torch.ones_like(ids))
    return torch.cumsum(n[:local], 0).clamp(max=rows).to(torch.int32)


def _grouped_inputs(case, seed):
    """Rows as a norm leaves them and the experts' weights: (x, w) in bfloat16,
    or (codes, scales, codes, block scales)."""
    E, N, C, M = _sizes(case)
    g = _generator(seed, 3)
    x = torch.randn((M, C), generator=g, device="cuda")
    fp8 = case["op"] == "mm8"
    w = torch.empty((E, N, C), dtype=FP8 if fp8 else torch.bfloat16, device="cuda")
    ws = torch.empty((E, -(-N // GROUP), -(-C // GROUP)), device="cuda")
    for e in range(E):
        v = torch.randn((N, C), generator=g, device="cuda") * WEIGHT_STD
        if fp8:
            w[e], ws[e] = _quantize_blocks(v)
        else:
            w[e] = v
    return (*_quantize_rows(x), w, ws) if fp8 else (x.to(torch.bfloat16), w)


def prepare(case, seed):
    """What the program has before the call: activations, weights, row ends."""
    if case["op"] in ("norm", "norm8"):
        x, r, w = _norm_inputs(case, seed)
        return {"op": case["op"], "x": x, "residual": r, "w": w}
    if case["op"] == "silu8":
        return {"op": "silu8", "h": _silu_inputs(case, seed)}
    return {"op": case["op"], "in": _grouped_inputs(case, seed), "ends": _ends(case, seed),
            "dtype": DTYPES[case["dtype"]]}


# ---------------------------------------------------------------------------
# The operators
# ---------------------------------------------------------------------------


def _rms(x, residual, w):
    """The normalised rows in float32 and the new residual."""
    if residual is not None:
        residual = (x.to(torch.float32) + residual.to(torch.float32)).to(residual.dtype)
        x = residual
    v = x.to(torch.float32)
    y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPS) * w.to(torch.float32)
    return y, residual


def _product(x, w_of, ends, N, dtype):
    """The grouped product in float32: rows padded to the longest of the groups
    in use, one batched product over these."""
    M, C = x.shape
    row = torch.arange(M, device=x.device)
    e = torch.searchsorted(ends.long(), row, right=True)
    live = torch.nonzero(e < ends.numel()).reshape(-1)
    y = torch.zeros((M, N), device=x.device)
    used, u = torch.unique(e[live], return_inverse=True)
    if used.numel():
        n = torch.bincount(u, minlength=used.numel())
        place = torch.arange(u.numel(), device=x.device) - (torch.cumsum(n, 0) - n)[u]
        xs = torch.zeros((used.numel(), int(n.max()), C), device=x.device)
        xs[u, place] = x[live]
        y[live] = torch.bmm(xs, w_of(used).transpose(1, 2))[u, place]
    return y.to(dtype)


def run(state):
    op = state["op"]
    if own:
        from wisp.integrations.vllm import grouped_mm as gm
        from wisp.integrations.vllm import rows_fp8 as rows
        if op == "norm":
            return rows.add_rms_norm(state["x"], state["w"], EPS, state["residual"])
        if op == "norm8":
            return rows.add_rms_norm_fp8(state["x"], state["w"], EPS, state["residual"])
        if op == "silu8":
            return rows.silu_mul_fp8(state["h"])
        if op == "mm":
            return gm.grouped_mm(*state["in"], state["ends"], dtype=state["dtype"])
        return gm.grouped_mm_fp8(*state["in"], state["ends"])
    if op in ("norm", "norm8"):
        y, r = _rms(state["x"], state["residual"], state["w"])
        return (y.to(state["x"].dtype), r) if op == "norm" else (*_quantize_rows(y), r)
    if op == "silu8":
        gate, up = state["h"].to(torch.float32).chunk(2, dim=1)
        return _quantize_rows(gate / (1.0 + torch.exp(-gate)) * up)
    if op == "mm":
        x, w = state["in"]
        return _product(x.to(torch.float32), lambda used: w[used].to(torch.float32),
                        state["ends"], w.shape[1], state["dtype"])
    q, s, w, ws = state["in"]
    N, C = w.shape[1:]
    x = q.to(torch.float32) * s.repeat_interleave(GROUP, dim=1)[:, :C]
    bits = w.view(torch.uint8)
    return _product(x, lambda used: bits[used].view(FP8).to(torch.float32)
                    * _spread(ws[used], N, C), state["ends"], N, state["dtype"])


# ---------------------------------------------------------------------------
# Cost and accuracy
# ---------------------------------------------------------------------------


def work(case):
    """Rows in and out once each; for the products the weights of the experts
    in use (their expected number), the rows of the groups, and all of out."""
    if case["op"] in ("norm", "norm8"):
        n, wide = case["rows"] * case["cols"], 2 if case["dtype"] == "bf16" else 4
        scales = 4 * case["rows"] * -(-case["cols"] // GROUP)
        out = n * wide if case["op"] == "norm" else n + scales
        return {"bytes": n * wide * (3 if case["residual"] else 1) + out + wide * case["cols"],
                "flops": 6 * n}
    if case["op"] == "silu8":
        n = case["rows"] * case["inter"]
        return {"bytes": 5 * n + 4 * case["rows"] * -(-case["inter"] // GROUP), "flops": 8 * n}
    _, _, E, K = LAYERS[case["layer"]]
    local, N, C, M = _sizes(case)
    rows = case["tokens"] * K // case["ranks"]
    experts = local * (1.0 - (1.0 - K / E) ** case["tokens"])
    wide = 1 if case["op"] == "mm8" else 2
    scales = 0 if wide == 2 else 4 * -(-C // GROUP) * (rows + experts * -(-N // GROUP))
    return {"bytes": int(wide * C * (rows + experts * N) + scales
                         + M * N * (2 if case["dtype"] == "bf16" else 4)),
            "flops": 2 * rows * N * C}


def _e4m3(a):
    """The float64 values nearest to ``a`` among those of e4m3 (4 significant
    bits down to 2^-6, steps of 2^-9 below; ties to even), saturating at 448."""
    e = torch.where(a == 0, -6, torch.frexp(a).exponent - 1).clamp(min=-6)
    step = ((e.to(torch.int64) - 3 + 1023) << 52).view(torch.float64)
    return (torch.round(a / step) * step).clamp(-TOP, TOP)


def _exact_rows(y):
    """The values of the codes and the scales of the float64 rows ``y``."""
    codes, scales = torch.empty_like(y), []
    for c in range(0, y.shape[1], GROUP):
        part = y[:, c:c + GROUP]
        s = part.abs().amax(dim=1, keepdim=True).clamp(min=LEAST) / TOP
        codes[:, c:c + GROUP] = _e4m3(part / s)
        scales.append(s)
    return codes, torch.cat(scales, dim=1)


def exact(case, seed):
    if case["op"] in ("norm", "norm8"):
        x, r, w = _norm_inputs(case, seed)
        if r is not None:
            r = (x.to(torch.float64) + r.to(torch.float64)).to(r.dtype)
            x = r
        v = x.to(torch.float64)
        y = v * torch.rsqrt(torch.mean(v ** 2, dim=1, keepdim=True) + EPS) * w.to(torch.float64)
        r = None if r is None else r.to(torch.float64)
        return (y, r) if case["op"] == "norm" else (*_exact_rows(y), r)
    if case["op"] == "silu8":
        gate, up = _silu_inputs(case, seed).to(torch.float64).split(case["inter"], dim=1)
        return _exact_rows(gate * torch.sigmoid(gate) * up)
    E, N, C, M = _sizes(case)
    given = _grouped_inputs(case, seed)
    out = torch.zeros((M, N), dtype=torch.float64, device="cuda")
    first = 0
    for e, end in enumerate(_ends(case, seed).tolist()):
        if end > first:
            part = slice(first, end)
            if case["op"] == "mm":
                x, w = given[0][part].to(torch.float64), given[1][e].to(torch.float64)
            else:
                q, s, w, ws = given
                x, w = q[part].to(torch.float64), w[e].to(torch.float64)
                block = torch.arange(N, device="cuda") // GROUP
                for c in range(-(-C // GROUP)):
                    at = slice(c * GROUP, (c + 1) * GROUP)
                    x[:, at] *= s[part, c:c + 1].to(torch.float64)
                    w[:, at] *= ws[e, block, c:c + 1].to(torch.float64)
            out[part] = x @ w.t()
        first = max(first, end)
    return out
