"""Performance cases of the MXFP4 operators: quantising weights to 4-bit
microscaled floating point and reading them back, the SwiGLU experts over such
weights, and the whole MoE layer over them from router logits.

MXFP4: a row's values in blocks of 32, each a 4-bit E2M1 code (two to a byte,
the earlier value in the low half) and one E8M0 scale byte s per block; a value
is E2M1(code) * 2^(s - 127).

With ``own`` false, ``run`` computes the operators from elementary torch
operations in float32, rounded once at the end; with ``own`` true it calls
``wisp.integrations.vllm.fused_moe_mxfp4``.
"""
from __future__ import annotations

import math

import torch

own = False

WEIGHT_STD = 0.02
BLOCK = 32
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

# hidden, inter, experts, top_k
LAYERS = {
    "toy": (512, 256, 16, 2),
    "odd": (1056, 352, 24, 3),
    "qwen3": (2048, 768, 128, 8),
    "mixtral": (4096, 14336, 8, 2),
}


def _matrix(name, op, rows, cols, dtype):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "dtype": dtype}


def _moe(name, op, layer, tokens, logits="bf16", missing=0.0):
    return {"name": name, "op": op, "layer": layer, "tokens": tokens, "logits": logits,
            "missing": missing}


def listed():
    return [
        # Quantised and read back, as a program does that looks at what 4 bits
        # do to a weight: one small float32 matrix (launches are all there
        # is), and the gate/up rows of 16 Qwen3 experts.
        _matrix("roundtrip-toy-f32", "roundtrip", 512, 512, "f32"),
        _matrix("roundtrip-qwen3-bf16", "roundtrip", 16 * 1536, 2048, "bf16"),
        # Reading back: an odd float32 one, and a Mixtral expert's gate/up rows.
        _matrix("dequantize-odd-f32", "dequantize", 333, 1376, "f32"),
        _matrix("dequantize-mixtral-bf16", "dequantize", 28672, 4096, "bf16"),
        # One token through a small layer, and bs=1 generation.
        _moe("layer-toy-1", "layer", "toy", 1, "f32"),
        _moe("layer-qwen3-1", "layer", "qwen3", 1, "f32"),
        # A few users of a layer with few large experts.
        _moe("layer-mixtral-6", "layer", "mixtral", 6),
        # Experts for given slots: batched generation; odd sizes, with a fifth
        # of the pairs on experts that are not here.
        _moe("experts-qwen3-32", "experts", "qwen3", 32),
        _moe("experts-odd-77-missing", "experts", "odd", 77, missing=0.2),
        # Prompt chunks: an ordinary one, the largest, one of few large experts.
        _moe("layer-qwen3-512", "layer", "qwen3", 512),
        _moe("experts-qwen3-8192", "experts", "qwen3", 8192),
        _moe("layer-mixtral-1000", "layer", "mixtral", 1000),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: matrices of other sizes, the same
    layers at other token counts."""
    op = rng.choice(["roundtrip", "dequantize", "experts", "experts", "layer", "layer"])
    if op in ("roundtrip", "dequantize"):
        cols = BLOCK * _log_int(rng, 1, 448)
        most = 28672 * 4096 // cols
        c = _matrix("", op, _log_int(rng, min(64, most), min(65536, most)), cols,
                    rng.choice(["bf16", "f32"]))
    else:
        layer = rng.choice(["toy", "odd", "qwen3", "qwen3", "qwen3", "mixtral"])
        most = {"toy": 4096, "odd": 4096, "qwen3": 8192, "mixtral": 1000}[layer]
        c = _moe("", op, layer, _log_int(rng, 1, most), rng.choice(["bf16", "f32"]),
                 round(rng.uniform(0.0, 0.5), 2) if op == "experts" and rng.random() < 0.3 else 0.0)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _scale_value(s):
    """2^(s - 127) in float32 of scale bytes s; 255 is NaN."""
    b = s.to(torch.int32)
    v = torch.where(b == 0, torch.full_like(b, 1 << 22), b << 23).view(torch.float32)
    return torch.where(b == 255, torch.full_like(v, float("nan")), v)


def _quantize(v):
    """``v [..., C]`` -> codes ``[..., C / 2]``, scale bytes ``[..., C / 32]``:
    the block's scale is 2^(floor(log2 max|v|) - 2), values are rounded to the
    nearest code (ties to the even one) and saturate at 6."""
    b = v.to(torch.float32).reshape(*v.shape[:-1], -1, BLOCK)
    top = b.abs().amax(dim=-1)
    s = ((top.view(torch.int32) >> 23) - 2).clamp(0, 254)
    a = (b / _scale_value(s)[..., None]).abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5.0)) + (torch.signbit(b).to(torch.uint8) << 3)
    code = code.to(torch.uint8).reshape(*v.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), s.to(torch.uint8)


def _dequantize(codes, scales):
    """The float32 values of codes ``[..., C / 2]`` and scales ``[..., C / 32]``."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    pair = torch.stack((codes & 15, codes >> 4), dim=-1).to(torch.int32)
    v = table[pair].reshape(*scales.shape, BLOCK) * _scale_value(scales)[..., None]
    return v.reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def _generator(seed, which):
    return torch.Generator(device="cuda").manual_seed(4 * seed + which)


def _weight(case, seed):
    """A weight matrix: rows of unequal norm, in the case's type."""
    g = _generator(seed, 0)
    v = torch.randn((case["rows"], case["cols"]), generator=g, device="cuda") * WEIGHT_STD
    v *= torch.exp(0.5 * torch.randn((case["rows"], 1), generator=g, device="cuda"))
    return v.to(DTYPES[case["dtype"]])


def _expert_weights(case, seed):
    """w13 ``[E, 2I, H]`` and w2 ``[E, H, I]`` as (codes, scales) pairs."""
    H, I, E, _ = LAYERS[case["layer"]]
    g = _generator(seed, 1)
    out = []
    for rows, cols in ((2 * I, H), (H, I)):
        q = torch.empty((E, rows, cols // 2), dtype=torch.uint8, device="cuda")
        s = torch.empty((E, rows, cols // BLOCK), dtype=torch.uint8, device="cuda")
        for e in range(E):
            q[e], s[e] = _quantize(torch.randn((rows, cols), generator=g, device="cuda")
                                   * WEIGHT_STD)
        out += [q, s]
    return out


def _inputs(case, seed):
    """Activations ``[T, H]`` as a normalisation leaves them, logits ``[T, E]``."""
    H, _, E, _ = LAYERS[case["layer"]]
    g = _generator(seed, 2)
    x = torch.randn((case["tokens"], H), generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.randn((case["tokens"], E), generator=g, device="cuda")
    return x, logits.to(DTYPES[case["logits"]])


def _slots(case, seed, logits):
    """Routing weights and slots for the experts' own call: top-k of the
    logits, some pairs (a whole token's now and then) without a slot."""
    w, ids = _route(logits, LAYERS[case["layer"]][3])
    if case["missing"]:
        g = _generator(seed, 3)
        gone = torch.rand(ids.shape, generator=g, device="cuda") < case["missing"]
        ids = torch.where(gone, torch.full_like(ids, -1), ids)
    return w, ids


def prepare(case, seed):
    """The weights, the plain or quantised ones, and the call's inputs."""
    if case["op"] == "roundtrip":
        return {"op": "roundtrip", "v": _weight(case, seed)}
    if case["op"] == "dequantize":
        q, s = _quantize(_weight(case, seed))
        return {"op": "dequantize", "q": q, "s": s, "dtype": DTYPES[case["dtype"]]}
    x, logits = _inputs(case, seed)
    q13, s13, q2, s2 = _expert_weights(case, seed)
    state = {"op": case["op"], "x": x, "k": LAYERS[case["layer"]][3], "q13": q13, "s13": s13,
             "q2": q2, "s2": s2}
    if case["op"] == "layer":
        state["logits"] = logits
    else:
        state["w"], state["slots"] = _slots(case, seed, logits)
    return state


# ---------------------------------------------------------------------------
# The operators
# ---------------------------------------------------------------------------


def _route(logits, k):
    """Renormalised softmax weights float32 and ids int32 ``[T, k]`` of the
    largest logits, ties to the lower id."""
    v = logits.to(torch.float32)
    ids = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :k]
    p = torch.exp(v - v.amax(dim=1, keepdim=True))
    w = p.gather(1, ids)
    return w / w.sum(dim=1, keepdim=True), ids.to(torch.int32)


def _experts(x, w, slots, q13, s13, q2, s2):
    """SwiGLU experts of the pairs that have a slot, in float32: the pairs
    sorted by expert, padded to the longest list, two batched products over
    the experts in use."""
    T, K = slots.shape
    H, I = x.shape[1], 2 * q2.shape[2]
    flat = slots.reshape(-1).long()
    pairs = torch.nonzero(flat >= 0).reshape(-1)
    y = torch.zeros((T * K, H), device=x.device)
    used, e = torch.unique(flat[pairs], return_inverse=True)
    if used.numel():
        e, order = torch.sort(e, stable=True)
        pairs = pairs[order]
        n = torch.bincount(e, minlength=used.numel())
        place = torch.arange(e.numel(), device=x.device) - (torch.cumsum(n, 0) - n)[e]
        xs = torch.zeros((used.numel(), int(n.max()), H), device=x.device)
        xs[e, place] = x[pairs // K].to(torch.float32)
        h = torch.bmm(xs, _dequantize(q13[used], s13[used]).transpose(1, 2))
        gate, up = h[..., :I], h[..., I:]
        act = gate / (1.0 + torch.exp(-gate)) * up
        y[pairs] = torch.bmm(act, _dequantize(q2[used], s2[used]).transpose(1, 2))[e, place]
    return (y.view(T, K, H) * w[..., None]).sum(dim=1).to(torch.bfloat16)


def run(state):
    op = state["op"]
    if own:
        from wisp.integrations.vllm import fused_moe_mxfp4 as mx
        if op == "roundtrip":
            return mx.dequantize_mxfp4(*mx.quantize_mxfp4(state["v"]), state["v"].dtype)
        if op == "dequantize":
            return mx.dequantize_mxfp4(state["q"], state["s"], state["dtype"])
        weights = state["q13"], state["q2"], state["s13"], state["s2"]
        if op == "experts":
            return mx.experts_mxfp4(state["x"], state["w"], state["slots"], *weights)
        return mx.route_and_experts_mxfp4(state["x"], state["logits"], state["k"], True, *weights)
    if op == "roundtrip":
        return _dequantize(*_quantize(state["v"])).to(state["v"].dtype)
    if op == "dequantize":
        return _dequantize(state["q"], state["s"]).to(state["dtype"])
    w, slots = (state["w"], state["slots"]) if op == "experts" else \
        _route(state["logits"], state["k"])
    return _experts(state["x"], w, slots, state["q13"], state["s13"], state["q2"], state["s2"])


# ---------------------------------------------------------------------------
# Cost and accuracy
# ---------------------------------------------------------------------------


def work(case):
    """A matrix in and out (the codes between the two calls of a round trip
    are not counted); for the experts x, out, logits or slots, and the weights
    of the experts the call routes to (their expected number), once each."""
    if case["op"] in ("roundtrip", "dequantize"):
        n = case["rows"] * case["cols"]
        wide = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": n * wide + (n * wide if case["op"] == "roundtrip" else n * 17 // 32),
                "flops": n}
    H, I, E, K = LAYERS[case["layer"]]
    T, share = case["tokens"], 1.0 - case["missing"]
    experts = E * (1.0 - (1.0 - share * K / E) ** T)
    routing = T * K * 8 if case["op"] == "experts" else \
        T * E * (2 if case["logits"] == "bf16" else 4)
    return {"bytes": int(experts * 3 * H * I * 17 // 32 + 4 * T * H + routing),
            "flops": int(share * T * K * 6 * H * I)}


def _power(e):
    """2^e in float64 of whole numbers e, made from its bits: a power function
    is off by its last bit here and there, and would break ties."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_values(q, s):
    """Float64 values of the codes and scales, one code half at a time."""
    v = torch.empty((*q.shape[:-1], 2 * q.shape[-1]), dtype=torch.float64, device=q.device)
    for half, shift in ((0, 0), (1, 4)):
        c = (q >> shift) & 15
        e, m = (c >> 1) & 3, (c & 1).to(torch.float64)
        size = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * _power(e.to(torch.int64) - 1))
        v[..., half::2] = torch.where(c >= 8, -size, size)
    return v * _power(s.to(torch.int64) - 127).repeat_interleave(BLOCK, dim=-1)


def _nearest(v):
    """Float64 values of ``v`` in MXFP4, from the definition: the nearest of
    the eight magnitudes, of two equally near ones the one of even code."""
    b = v.to(torch.float64).reshape(v.shape[0], -1, BLOCK)
    top = b.abs().amax(dim=2, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(-127, 127)
    scale = _power(e)
    a = b.abs() / scale
    best = torch.zeros_like(a)
    for i in (2, 4, 6, 1, 3, 5, 7):  # an odd code has to be strictly nearer
        m = MAGNITUDES[i]
        near, far = (a - m).abs(), (a - best).abs()
        best = torch.where(near < far, torch.full_like(a, m), best)
        if i in (2, 4, 6):
            best = torch.where(near == far, torch.full_like(a, m), best)
    return (torch.sign(b) * best * scale).reshape(v.shape)


def exact(case, seed):
    if case["op"] == "roundtrip":
        return _nearest(_weight(case, seed))
    if case["op"] == "dequantize":
        return _exact_values(*_quantize(_weight(case, seed)))
    H, I, E, K = LAYERS[case["layer"]]
    x, logits = _inputs(case, seed)
    q13, s13, q2, s2 = _expert_weights(case, seed)
    if case["op"] == "experts":
        w, ids = _slots(case, seed, logits)
        w = w.to(torch.float64)
    else:
        p = torch.softmax(logits.to(torch.float64), dim=1)
        ids = torch.sort(logits.to(torch.float64), dim=1, descending=True,
                         stable=True).indices[:, :K]
        w = p.gather(1, ids)
        w = w / w.sum(dim=1, keepdim=True)
    out = torch.zeros((case["tokens"], H), dtype=torch.float64, device="cuda")
    for e in range(E):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        h = x[t].to(torch.float64) @ _exact_values(q13[e], s13[e]).t()
        act = torch.nn.functional.silu(h[:, :I]) * h[:, I:]
        out.index_add_(0, t, (act @ _exact_values(q2[e], s2[e]).t()) * w[t, k][:, None])
    return out
