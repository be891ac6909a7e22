"""MXFP4 operators on the GPU against the float64 oracle: quantising and reading
back bit for bit, the experts and the whole layer within the bound that float32
sums and two bf16 roundings allow (derived in ``oracle.mxfp4.experts``), at
sizes, masks and values where they can go wrong."""
import functools

import numpy as np
import pytest
import torch

from oracle import mxfp4 as O
from oracle.moe import route
from wisp.integrations.vllm import fused_moe_mxfp4 as mx

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


# ---------------------------------------------------------------------------
# Quantising and reading back
# ---------------------------------------------------------------------------


def _matrix(rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    v = torch.randn((rows, cols), generator=g) * torch.exp(3 * torch.randn((rows, 1), generator=g))
    v[torch.rand(v.shape, generator=g) < 0.05] = 0.0
    v[torch.rand(v.shape, generator=g) < 0.02] *= -0.0
    return v


def _check_quant(v):
    q, s = mx.quantize_mxfp4(v.to(DEV))
    wq, ws = O.quantize(v.float().numpy())
    assert np.array_equal(s.cpu().numpy(), ws)
    assert np.array_equal(q.cpu().numpy(), wq)
    return q, s


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 64), (3, 96), (7, 1056), (64, 128), (257, 160),
                                       (33, 4096)])
def test_quantize_is_exact(rows, cols, dtype):
    _check_quant(_matrix(rows, cols, rows + cols).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_special_blocks(dtype):
    v = torch.zeros((16, 64), dtype=dtype)
    for i, x in enumerate((0.0, -0.0, 2.0 ** -126, 2.0 ** -133, -(2.0 ** -124), 3.3e38, -3.3e38,
                           float("inf"), float("-inf"), float("nan"), 6.0, 7.9, 5.0, -2.5, 0.25)):
        v[i, (7 * i) % 64] = x
        v[i, (7 * i + 3) % 64] = x / 3
    _check_quant(v)


def test_quantize_every_bf16_value():
    """Every finite bf16 magnitude beside block maxima that put it at, above
    and far below the top of the block."""
    bits = torch.arange(0x7f80, dtype=torch.int32)
    a = (bits << 16).view(torch.float32)
    rows = []
    for up in (0, 1, 3, 6):
        top = torch.clamp(a.double() * 2.0 ** up, max=3.0e38).to(torch.bfloat16)
        row = torch.zeros((a.numel(), 32), dtype=torch.bfloat16)
        row[:, 0] = a.to(torch.bfloat16)
        row[:, 17] = -a.to(torch.bfloat16)
        row[:, 31] = top
        rows.append(row)
    _check_quant(torch.cat(rows))


def test_quantize_ties():
    v = torch.tensor([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5.0] + [0] * 24)
    m = torch.stack([v * 2.0 ** e for e in range(-130, 124)])
    _check_quant(torch.cat([m, -m]))


def test_quantize_shapes_and_strides():
    v = _matrix(24, 256, 5)
    q, s = _check_quant(v)
    a, b = mx.quantize_mxfp4(v.view(2, 3, 4, 256).to(DEV))
    assert a.shape == (2, 3, 4, 128) and b.shape == (2, 3, 4, 8)
    assert torch.equal(a.view(24, 128), q) and torch.equal(b.view(24, 8), s)
    wide = torch.zeros((24, 512), device=DEV)
    wide[:, 8:264] = v.to(DEV)
    a, b = mx.quantize_mxfp4(wide[:, 8:264])
    assert torch.equal(a, q) and torch.equal(b, s)
    a, b = mx.quantize_mxfp4(wide.view(-1)[9:9 + 32])  # not 16-byte aligned
    assert torch.equal(a, mx.quantize_mxfp4(wide.view(-1)[9:9 + 32].clone())[0])
    a, b = mx.quantize_mxfp4(torch.empty((0, 64), device=DEV))
    assert a.shape == (0, 32) and b.shape == (0, 2)
    assert mx.dequantize_mxfp4(a, b).shape == (0, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dequantize_every_code_and_scale(dtype):
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 16)
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    got = mx.dequantize_mxfp4(codes.to(DEV), scales.to(DEV), dtype).cpu()
    with np.errstate(over="ignore", invalid="ignore"):
        want = torch.from_numpy(O.dequantize(codes.numpy(), scales.numpy())).to(dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isnan(want[255]).all()
    assert torch.equal(torch.nan_to_num(got, nan=1.0), torch.nan_to_num(want, nan=1.0))


@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 96), (333, 1376), (70, 4096)])
def test_dequantize_sizes_and_strides(rows, cols):
    q, s = O.quantize(_matrix(rows, cols, 9).numpy())
    tq, ts = torch.from_numpy(q).to(DEV), torch.from_numpy(s).to(DEV)
    want = torch.from_numpy(O.dequantize(q, s)).float()
    assert torch.equal(mx.dequantize_mxfp4(tq, ts, torch.float32).cpu(), want)
    pad = torch.zeros((rows, cols // 2 + 2), dtype=torch.uint8, device=DEV)
    pad[:, 1:-1] = tq
    assert torch.equal(mx.dequantize_mxfp4(pad[:, 1:-1], ts, torch.float32).cpu(), want)
    flat = torch.zeros(cols // 2 + 1, dtype=torch.uint8, device=DEV)
    flat[1:] = tq[0]
    assert torch.equal(mx.dequantize_mxfp4(flat[1:], ts[0], torch.float32).cpu(), want[0])


def test_quantize_refusals():
    for bad in (torch.zeros((2, 48), device=DEV), torch.zeros((), device=DEV)):
        with pytest.raises(ValueError):
            mx.quantize_mxfp4(bad)
    with pytest.raises(NotImplementedError):
        mx.quantize_mxfp4(torch.zeros((2, 64), device=DEV, dtype=torch.float16))
    q, s = mx.quantize_mxfp4(torch.zeros((2, 64), device=DEV))
    for a, b in ((q, s[:1]), (q.float(), s), (q, s.cpu()), (q[:, :24], s)):
        with pytest.raises(ValueError):
            mx.dequantize_mxfp4(a, b)
    with pytest.raises(NotImplementedError):
        mx.dequantize_mxfp4(q, s, torch.float16)


# ---------------------------------------------------------------------------
# Experts
# ---------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _weights(E, H, I, seed, std=0.05):
    rng = np.random.default_rng(seed)
    out = []
    for shape in ((E, 2 * I, H), (E, H, I)):
        w = rng.standard_normal(shape).astype(np.float32) * std
        w *= 2.0 ** rng.integers(-3, 4, (*shape[:2], 1)).astype(np.float32)
        out += O.quantize(w)
    return tuple(out)  # w13, s13, w2, s2


def _routing(T, E, K, seed):
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.permutation(E)[:K] for _ in range(T)]).astype(np.int32).reshape(T, K)
    return ids, rng.uniform(0.05, 1.0, (T, K)).astype(np.float32)


def _x(T, H, seed):
    return torch.randn((T, H), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def _dev(w):
    return [torch.from_numpy(np.ascontiguousarray(a)).to(DEV) for a in w]


def _run(x, w, slots, weights, **kw):
    w13, s13, w2, s2 = _dev(weights) if isinstance(weights[0], np.ndarray) else weights
    return mx.experts_mxfp4(x.to(DEV), torch.as_tensor(w).to(DEV),
                            torch.as_tensor(np.asarray(slots)).to(DEV), w13, w2, s13, s2, **kw)


def _close(got, x, w, slots, weights):
    want, bound = O.experts(x.double().numpy(), w, slots, *weights)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound).all(), float((err / bound).max())


SHAPES = [  # T, H, I, E, K
    (1, 32, 32, 1, 1), (1, 512, 256, 16, 2), (1, 2048, 768, 16, 8), (2, 96, 160, 5, 3),
    (3, 1056, 352, 24, 3), (5, 64, 96, 70, 20), (8, 2048, 768, 16, 8), (16, 512, 256, 16, 8),
    (17, 256, 64, 5, 5), (33, 160, 128, 4, 1), (70, 160, 96, 4, 2), (77, 1056, 352, 24, 3),
    (200, 128, 192, 3, 1), (300, 512, 256, 16, 2), (600, 256, 416, 2, 2), (1100, 384, 288, 3, 2),
    (12, 64, 4160, 6, 4), (20, 96, 3104, 4, 4), (40, 128, 9216, 3, 2), (130, 128, 128, 2, 1),
    (200, 256, 640, 3, 2), (401, 512, 128, 2, 2), (1300, 256, 384, 5, 1),
    (250, 256, 512, 4, 1), (250, 160, 96, 4, 1), (330, 256, 512, 4, 1), (330, 160, 96, 4, 1),
    (280, 128, 12800, 2, 1), (350, 128, 12800, 2, 1), (280, 25600, 128, 2, 1),
    (350, 25600, 128, 2, 1),
]


@pytest.mark.parametrize("T,H,I,E,K", SHAPES)
def test_experts_match_the_oracle(T, H, I, E, K):
    weights = _weights(E, H, I, T)
    ids, w = _routing(T, E, K, T + 1)
    x = _x(T, H, T + 2)
    _close(_run(x, w, ids, weights), x, w, ids, weights)


@pytest.mark.parametrize("T,H,I,E,K", [(13, 64, 6400, 4, 2), (20, 96, 6208, 3, 1),
                                       (30, 32, 8448, 2, 2), (13, 64, 14336, 4, 2)])
def test_experts_of_a_long_inner_range(T, H, I, E, K):
    """w2's k range does not split evenly; a call of NaNs before leaves NaNs
    wherever a kernel keeps its operands."""
    weights = _weights(E, H, I, T)
    dev = _dev(weights)
    ids, w = _routing(T, E, K, T + 1)
    x = _x(T, H, T + 2)
    assert torch.isnan(_run(torch.full_like(x, float("nan")), w, ids, dev)).all()
    _close(_run(x, w, ids, dev), x, w, ids, weights)


@pytest.mark.parametrize("T", [1, 20, 400])
def test_experts_of_large_gates(T):
    """Gates from -1500 to 1500: the exponential of their negative overflows."""
    E, H, I, K = 2, 256, 128, 1
    weights = _weights(E, H, I, 21, std=10.0)
    ids, w = _routing(T, E, K, 22)
    x = _x(T, H, 23)
    g = x[:1].double().numpy() @ O.dequantize(weights[0][ids[0, 0]], weights[1][ids[0, 0]])[:I].T
    assert (g < -95).any() and (g > 95).any()
    _close(_run(x, w, ids, weights), x, w, ids, weights)


@pytest.mark.parametrize("H,I", [(32, 64), (128, 128)])
def test_experts_of_many_tokens(H, I):
    """More tokens than 16 bits count: the last rows are those of a small call."""
    T, E, K = 70001, 3, 2
    weights = _weights(E, H, I, 8)
    dev = _dev(weights)
    ids, w = _routing(T, E, K, 9)
    x = _x(T, H, 10)
    got = _run(x, w, ids, dev)
    for part in (slice(0, 20), slice(65530, 65550), slice(T - 20, T)):
        assert torch.equal(got[part], _run(x[part], w[part], ids[part], dev))
        _close(got[part], x[part], w[part], ids[part], weights)


@pytest.mark.parametrize("T,H,I,E,K", [s for s in SHAPES if s[0] in (1, 3, 17, 77, 300)])
def test_experts_missing_slots(T, H, I, E, K):
    """Slots outside [0, E) contribute nothing, whole tokens without a slot
    are zero, and so is a call without any."""
    weights = _weights(E, H, I, T)
    ids, w = _routing(T, E, K, T + 1)
    x = _x(T, H, T + 2)
    rng = np.random.default_rng(3)
    slots = ids.copy()
    slots[rng.uniform(size=ids.shape) < 0.4] = -1
    slots[rng.uniform(size=ids.shape) < 0.1] = E
    slots[rng.uniform(size=ids.shape) < 0.1] = 2 ** 31 - 1
    slots[rng.integers(T)] = -1
    seen = np.where((slots < 0) | (slots >= E), -1, slots)
    got = _run(x, w, slots, weights)
    _close(got, x, w, seen, weights)
    assert not got[torch.from_numpy((seen < 0).all(axis=1)).to(DEV)].any()
    assert not _run(x, w, np.full_like(ids, -1), weights).any()


@pytest.mark.parametrize("T", [1, 4, 24])
def test_experts_same_expert_twice(T):
    E, H, I, K = 3, 96, 64, 5
    weights = _weights(E, H, I, 1)
    rng = np.random.default_rng(4)
    slots = rng.integers(0, E, (T, K)).astype(np.int32)
    slots[0] = 2
    w = rng.uniform(0.05, 1.0, (T, K)).astype(np.float32)
    x = _x(T, H, 5)
    _close(_run(x, w, slots, weights), x, w, slots, weights)


@pytest.mark.parametrize("T", [1, 5, 40])
def test_experts_special_values_stay_where_they_are(T):
    """A NaN scale reaches the tokens of its expert only, an infinite or NaN
    activation its own token only; every other row keeps its bytes."""
    E, H, I, K = 6, 160, 96, 2
    weights = _dev(_weights(E, H, I, 2))
    ids, w = _routing(T, E, K, 6)
    x = _x(T, H, 7)
    base = _run(x, w, ids, weights)
    assert torch.isfinite(base).all()
    for which in (1, 3):
        bad = [a.clone() for a in weights]
        bad[which][1, 3, -1] = 255
        got = _run(x, w, ids, bad)
        hit = torch.from_numpy((ids == 1).any(axis=1)).to(DEV)
        assert torch.equal(got[~hit], base[~hit])
        if hit.any():
            assert torch.isnan(got[hit]).any(dim=1).all()
    for v in (float("inf"), float("nan")):
        y = x.clone()
        y[0, H - 1] = v
        got = _run(y, w, ids, weights)
        assert torch.equal(got[1:], base[1:]) and not torch.isfinite(got[0]).all()


def test_experts_smallest_and_largest_scales():
    """Weights below bf16's normal numbers, against activations that lift
    them, and scales near the top."""
    T, E, H, I, K = 3, 2, 64, 64, 2
    rng = np.random.default_rng(8)
    w13 = rng.integers(0, 256, (E, 2 * I, H // 2)).astype(np.uint8)
    w2 = rng.integers(0, 256, (E, H, I // 2)).astype(np.uint8)
    s13 = np.full((E, 2 * I, H // 32), 0, np.uint8)
    s2 = np.full((E, H, I // 32), 127, np.uint8)
    ids, w = _routing(T, E, K, 9)
    x = (_x(T, H, 10).double() * 2.0 ** 120).to(torch.bfloat16)
    weights = [w13, s13, w2, s2]
    _close(_run(x, w, ids, weights), x, w, ids, weights)
    weights = [w13, np.full_like(s13, 250), w2, s2]
    x = (_x(T, H, 10).double() * 2.0 ** -126).to(torch.bfloat16)
    _close(_run(x, w, ids, weights), x, w, ids, weights)


@pytest.mark.parametrize("T", [1, 6, 50])
def test_experts_slot_placement_and_strides(T):
    """The same experts at other slots, in a slab with other data between,
    and activations and routing with strides: the same bytes."""
    E, H, I, K = 7, 288, 96, 3
    weights = _weights(E, H, I, 3)
    ids, w = _routing(T, E, K, 11)
    x = _x(T, H, 12)
    base = _run(x, w, ids, weights)
    perm = np.random.default_rng(13).permutation(E)
    slab = 256 * (-(-sum(a[0].size for a in weights) // 256))
    buf = torch.full((E, slab), 255, dtype=torch.uint8, device=DEV)
    views, off = [], 0
    for i in (0, 2, 1, 3):
        a = weights[i]
        v = torch.as_strided(buf, a.shape, (slab, a.shape[2], 1), off)
        v.copy_(torch.from_numpy(a[perm]))
        views.append(v)
        off += a[0].size
    slots = np.argsort(perm)[ids].astype(np.int32)
    wide = torch.full((T, 2 * H), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, H:] = x.to(DEV)
    ws = torch.zeros((K, T), device=DEV)
    ws.copy_(torch.from_numpy(w.T.copy()))
    ss = torch.zeros((K, T), dtype=torch.int32, device=DEV)
    ss.copy_(torch.from_numpy(slots.T.copy()))
    out = torch.empty((T, H), dtype=torch.bfloat16, device=DEV)
    got = mx.experts_mxfp4(wide[:, H:], ws.t(), ss.t(), views[0], views[1], views[2], views[3],
                           out=out)
    assert got is out and torch.equal(got, base)


def test_experts_leave_their_surroundings_alone():
    T, E, H, I, K = 3, 4, 96, 64, 2
    weights = _weights(E, H, I, 4)
    ids, w = _routing(T, E, K, 14)
    big = torch.full((T + 2, H), 7.0, dtype=torch.bfloat16, device=DEV)
    _run(_x(T, H, 15), w, ids, weights, out=big[1:T + 1])
    assert (big[0] == 7).all() and (big[T + 1] == 7).all() and not (big[1:T + 1] == 7).all()


def test_experts_other_stream_and_graph():
    """On a side stream, and captured: two graphs of different sizes, replayed
    in turn with eager calls between, every replay equal to the eager result."""
    E, H, I, K = 16, 512, 256, 2
    weights = _dev(_weights(E, H, I, 5))
    sets = []
    for T in (1, 9, 40):
        ids, w = _routing(T, E, K, T)
        sets.append([_x(T, H, T).to(DEV), torch.from_numpy(w).to(DEV),
                     torch.from_numpy(ids).to(DEV)])
    w13, s13, w2, s2 = weights
    call = lambda a: mx.experts_mxfp4(a[0], a[1], a[2], w13, w2, s13, s2)  # noqa: E731
    eager = [call(a) for a in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [call(a) for a in sets]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graphs = []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = call(a)
        graphs.append((g, r))
    for n in range(3):
        for a in sets:
            a[0].mul_(-0.5)
        want = [call(a) for a in sets]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, r), b in zip(graphs, want):
            assert torch.equal(r, b)


@pytest.mark.parametrize("T,H,I,E,K", [(700, 256, 256, 6, 1), (30, 128, 2304, 4, 2)])
def test_layer_in_a_graph(T, H, I, E, K):
    """The block tiles, and w2's k range in parts, captured and replayed with
    eager calls between."""
    w13, s13, w2, s2 = _dev(_weights(E, H, I, 31))
    x, lg = _x(T, H, 32).to(DEV), torch.randn((T, E), device=DEV)
    call = lambda: mx.route_and_experts_mxfp4(x, lg, K, True, w13, w2, s13, s2)  # noqa: E731
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    for _ in range(3):
        x.mul_(-0.5)
        lg.copy_(lg.flip(1))
        want = call()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_experts_refusals():
    E, H, I, K, T = 4, 64, 32, 2, 3
    w13, s13, w2, s2 = _dev(_weights(E, H, I, 6))
    ids, w = _routing(T, E, K, 16)
    x, w, ids = _x(T, H, 17).to(DEV), torch.from_numpy(w).to(DEV), torch.from_numpy(ids).to(DEV)
    ok = dict(x=x, topk_w=w, slots=ids, w13=w13, w2=w2, s13=s13, s2=s2)
    for bad in (dict(slots=ids.long()), dict(slots=ids[:2]), dict(topk_w=w.double()),
                dict(topk_w=w[:, :1]), dict(w13=w13[:, :, :16]), dict(w13=w13.float()),
                dict(s13=s13[:3]), dict(s2=s2.cpu()), dict(slots=ids.cpu()),
                dict(w2=w2.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(out=torch.empty((T, H), device=DEV)), dict(x=x[0])):
        with pytest.raises(ValueError):
            mx.experts_mxfp4(**{**ok, **bad})
    with pytest.raises(NotImplementedError):
        mx.experts_mxfp4(**{**ok, "x": x.float()})
    assert mx.experts_mxfp4(**{**ok, "x": x[:0], "topk_w": w[:0], "slots": ids[:0]}).shape == (0, H)


# ---------------------------------------------------------------------------
# The whole layer
# ---------------------------------------------------------------------------


def _layer(x, logits, K, renorm, weights):
    w13, s13, w2, s2 = _dev(weights) if isinstance(weights[0], np.ndarray) else weights
    return mx.route_and_experts_mxfp4(x.to(DEV), logits.to(DEV), K, renorm, w13, w2, s13, s2)


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,I,E,K", SHAPES)
def test_layer_matches_the_oracle(T, H, I, E, K, dtype, renorm):
    """bf16 logits tie now and then: the lower id goes first."""
    weights = _weights(E, H, I, T)
    x = _x(T, H, T + 2)
    logits = torch.randn((T, E), generator=torch.Generator().manual_seed(T + 3)).to(dtype)
    w, ids = route(logits.float(), K, renorm)
    want, bound = O.experts(x.double().numpy(), w, ids, *weights)
    # the routing weights are float32: exponentials, a sum of E terms and two
    # divisions, each off by at most two steps
    bound = bound + (E + 16) * 2.0 ** -23 * (np.abs(want) + bound)
    err = np.abs(_layer(x, logits, K, renorm, weights).double().cpu().numpy() - want)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("T", [1, 7, 30])
def test_layer_is_routing_then_experts(T):
    """The layer's bytes are those of the experts on the router's weights and
    ids, with logits that tie, are infinite or lowest."""
    from wisp_amd import _lib
    E, H, I, K = 20, 256, 96, 4
    weights = _dev(_weights(E, H, I, 7))
    x = _x(T, H, 18).to(DEV)
    logits = torch.randn((T, E), generator=torch.Generator().manual_seed(19))
    logits[:, 3] = logits[:, 9] = 2.5
    logits[0, :10] = float("-inf")
    logits[-1, 5] = torch.finfo(torch.float32).min
    logits = logits.to(DEV)
    w = torch.empty((T, K), device=DEV)
    ids = torch.empty((T, K), dtype=torch.int32, device=DEV)
    _lib.check(_lib.lib().wisp_route_topk_softmax(
        logits.data_ptr(), _lib.WISP_F32, T, E, K, 1, w.data_ptr(), ids.data_ptr(), None,
        _lib.stream_handle()), "route")
    w13, s13, w2, s2 = weights
    assert torch.equal(_layer(x, logits, K, True, weights),
                       mx.experts_mxfp4(x, w, ids, w13, w2, s13, s2))


def test_layer_refusals():
    E, H, I, T = 4, 64, 32, 3
    w13, s13, w2, s2 = _dev(_weights(E, H, I, 8))
    x, lg = _x(T, H, 20).to(DEV), torch.zeros((T, E), device=DEV)
    for logits, k in ((lg[:, :3], 2), (lg, 0), (lg, 5), (lg.cpu(), 2)):
        with pytest.raises(ValueError):
            mx.route_and_experts_mxfp4(x, logits, k, True, w13, w2, s13, s2)
    assert mx.route_and_experts_mxfp4(x[:0], lg[:0], 2, True, w13, w2, s13, s2).shape == (0, H)


def test_a_whole_layer_from_bf16_weights():
    """Together, as they are used: weights quantised on the GPU, the layer on
    them, against the oracle on the values read back."""
    T, H, I, E, K = 6, 512, 256, 8, 2
    g = torch.Generator().manual_seed(21)
    a = (torch.randn((E, 2 * I, H), generator=g) * 0.02).to(torch.bfloat16).to(DEV)
    b = (torch.randn((E, H, I), generator=g) * 0.02).to(torch.bfloat16).to(DEV)
    (w13, s13), (w2, s2) = mx.quantize_mxfp4(a), mx.quantize_mxfp4(b)
    x = _x(T, H, 22)
    logits = torch.randn((T, E), generator=g)
    got = _layer(x, logits, K, True, [w13, s13, w2, s2])
    w, ids = route(logits, K)
    want, bound = O.experts(x.double().numpy(), w, ids, *[t.cpu().numpy() for t in (w13, s13, w2, s2)])
    bound = bound + (E + 16) * 2.0 ** -23 * (np.abs(want) + bound)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()
    # what four bits leave of a weight: half a step of at most a quarter of the
    # value and its scale, over the block maximum at least 4/6 of the top
    back = mx.dequantize_mxfp4(w13, s13).float() - a.float()
    assert float(back.norm() / a.float().norm()) < 0.25
