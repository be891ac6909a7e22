"""MXFP4 operators at the ends of their ranges: rows and activations of more
values than 32 bits count, the largest expert, many experts, and special
values, missing slots and extreme scales in every kernel."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import mxfp4 as O
from oracle.moe import route
from tests.test_gpu_mxfp4 import DEV, _close, _dev, _layer, _routing, _run, _weights, _x
from wisp.integrations.vllm import fused_moe_mxfp4 as mx
from wisp_amd import _lib

pytestmark = pytest.mark.gpu


def test_rows_longer_than_32_bits():
    """One row of 2^32 + 32 values: quantised and read back whole.  (Of each
    value's buffers the first stand in memory that held other bytes.)"""
    n = 2 ** 32 + 32
    for size in (n // 2, n // 32):
        torch.full((size,), 255, dtype=torch.uint8, device=DEV)
    w = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    for at, v in ((0, 3.0), (31, -0.5), (2 ** 31 - 1, 6.0), (2 ** 31, -1.5), (2 ** 32 - 1, 2.0),
                  (2 ** 32, -4.0), (n - 1, 1.0)):
        w[at] = v
    q, s = mx.quantize_mxfp4(w)
    assert q.shape == (n // 2,) and s.shape == (n // 32,)
    assert int((q != 0).sum()) == 7 and int((s != 0).sum()) == 5
    assert torch.equal(mx.dequantize_mxfp4(q, s), w)


# ---------------------------------------------------------------------------
# Experts, in each of their kernels: the two launches for a few tokens, the
# grouped GEMM with whole and odd stages, with w2's k range in parts, and the
# block tiles.  (T, H, I, E, K)
# ---------------------------------------------------------------------------

KERNELS = {
    "few": (5, 160, 96, 6, 2), "odd": (40, 160, 96, 6, 2), "whole": (40, 256, 512, 6, 2),
    "parts": (30, 128, 2304, 4, 2), "odd parts": (30, 160, 2144, 4, 2),
    "tiles 128": (200, 256, 512, 2, 1), "tiles 160": (280, 128, 12800, 2, 1),
    "tiles 192": (330, 256, 512, 4, 1), "many passes": (1500, 160, 96, 2, 1),
}


@pytest.mark.parametrize("name", KERNELS)
def test_special_values_stay_where_they_are(name):
    """A NaN scale, at a row's first, a middle and its last block, reaches the
    tokens of its expert only; an infinite or NaN activation its own token
    only.  Every other row keeps its bytes."""
    T, H, I, E, K = KERNELS[name]
    weights = _dev(_weights(E, H, I, 2))
    ids, w = _routing(T, E, K, 6)
    x = _x(T, H, 7)
    base = _run(x, w, ids, weights)
    assert torch.isfinite(base).all()
    e = int(ids[0, 0])
    hit = torch.from_numpy((ids == e).any(axis=1)).to(DEV)
    for which in (1, 3):
        for block in (0, weights[which].shape[2] // 2, -1):
            bad = [a.clone() for a in weights]
            bad[which][e, 3, block] = 255
            got = _run(x, w, ids, bad)
            assert torch.equal(got[~hit], base[~hit])
            assert torch.isnan(got[hit]).any(dim=1).all()
    for v in (float("inf"), float("-inf"), float("nan")):
        y = x.clone()
        at = sorted({0, T // 2, T - 1})
        for t, h in zip(at, (H - 1, 0, H // 2)):
            y[t, h] = v
        got = _run(y, w, ids, weights)
        keep = torch.ones(T, dtype=torch.bool)
        keep[at] = False
        assert torch.equal(got[keep.to(DEV)], base[keep.to(DEV)])
        assert not torch.isfinite(got[at]).all(dim=1).any()


@pytest.mark.parametrize("name", KERNELS)
def test_missing_slots_and_empty_experts(name):
    """Pairs without a slot, whole tokens of them, and experts without a pair."""
    T, H, I, E, K = KERNELS[name]
    weights = _weights(E, H, I, T)
    ids, w = _routing(T, E, K, T + 1)
    x = _x(T, H, T + 2)
    rng = np.random.default_rng(5)
    slots = np.where(ids == E - 1, 0, ids).astype(np.int32)  # (the last expert has no pair)
    slots[rng.uniform(size=ids.shape) < 0.3] = -1
    slots[rng.uniform(size=ids.shape) < 0.1] = E
    slots[T // 2] = -(2 ** 31)
    seen = np.where((slots < 0) | (slots >= E), -1, slots)
    got = _run(x, w, slots, weights)
    _close(got, x, w, seen, weights)
    assert not got[torch.from_numpy((seen < 0).all(axis=1)).to(DEV)].any()
    assert not _run(x, w, np.full_like(ids, -1), weights).any()
    one = np.full_like(ids, -1)
    one[T - 1, 0] = E - 1
    _close(_run(x, w, one, weights), x, w, one, weights)


@pytest.mark.parametrize("name", KERNELS)
def test_smallest_and_largest_scales(name):
    """Weights below bf16's normal numbers, against activations that lift
    them, and scales near the top."""
    T, H, I, E, K = KERNELS[name]
    rng = np.random.default_rng(8)
    w13 = rng.integers(0, 256, (E, 2 * I, H // 2)).astype(np.uint8)
    w2 = rng.integers(0, 256, (E, H, I // 2)).astype(np.uint8)
    s2 = np.full((E, H, I // 32), 127, np.uint8)
    ids, w = _routing(T, E, K, 9)
    for s, lift in ((0, 2.0 ** 120), (250, 2.0 ** -126)):
        weights = [w13, np.full((E, 2 * I, H // 32), s, np.uint8), w2, s2]
        x = (_x(T, H, 10).double() * lift).to(torch.bfloat16)
        _close(_run(x, w, ids, weights), x, w, ids, weights)


@pytest.mark.parametrize("T", [12, 20, 400])
def test_gates_at_the_end_of_the_exponential(T):
    """Gates down to -88.625, whose e^-g is near float32's largest and whose
    e^g is below its normal numbers, times up to 2^121: in float32 silu is a
    normal number there, and act up to 40."""
    H = I = 128
    gate, up, w2 = (np.zeros((1, n, m), np.float32) for n, m in ((I, H), (I, H), (H, I)))
    gate[:, :, 0], gate[:, :, 2] = 1.0, 0.125
    up[:, :, 1] = 2.0 ** (14 + np.arange(I) % 8)
    w2[0, np.arange(H), np.arange(I)] = 1.0
    weights = [*O.quantize(np.concatenate([gate, up], 1)), *O.quantize(w2)]
    assert np.array_equal(O.dequantize(*weights[:2]), np.concatenate([gate, up], 1))
    x = np.zeros((T, H), np.float32)
    t = np.arange(T)
    x[:, 0] = -88.0 + t % 10 * 0.5 * (t % 3 > 0)
    x[:, 2] = -(t // 3 % 6)
    x[:, 1] = np.where(t % 2, -(2.0 ** 100), 2.0 ** 100)
    g = x[:, 0] + 0.125 * x[:, 2]
    assert g.min() < -88.25 and (g > -86).any()
    x = torch.from_numpy(x).to(torch.bfloat16)
    slots, w = np.zeros((T, 1), np.int32), np.ones((T, 1), np.float32)
    _close(_run(x, w, slots, weights), x, w, slots, weights)


@pytest.mark.parametrize("T,H,I,E,K", [(2, 64, 32, 600, 3), (40, 64, 32, 600, 4),
                                       (900, 64, 96, 1000, 2)])
def test_more_slots_than_a_router_has(T, H, I, E, K):
    weights = _weights(E, H, I, T)
    ids, w = _routing(T, E, K, T + 1)
    x = _x(T, H, T + 2)
    _close(_run(x, w, ids, weights), x, w, ids, weights)


@pytest.mark.parametrize("empty", [False, True])
def test_block_tiles_of_many_experts(empty):
    """More experts than a wave has lanes, all in use, or runs of them not."""
    T, H, I, E = 8000, 128, 128, 90
    weights = _weights(E, H, I, 12)
    rng = np.random.default_rng(13)
    used = np.array([2, 3, 71, 72, 89]) if empty else np.arange(E)
    slots = used[rng.integers(0, len(used), (T, 1))].astype(np.int32)
    if empty:
        slots[rng.uniform(size=slots.shape) < 0.5] = -1
    w = rng.uniform(0.05, 1.0, (T, 1)).astype(np.float32)
    x = _x(T, H, 14)
    _close(_run(x, w, slots, weights), x, w, slots, weights)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,I,E,K", [(3, 64, 32, 130, 4), (2, 64, 32, 300, 8),
                                       (1, 32, 32, 512, 8), (1, 96, 64, 256, 64),
                                       (30, 64, 32, 512, 5)])
def test_layer_of_many_experts(T, H, I, E, K, dtype):
    weights = _weights(E, H, I, T)
    x = _x(T, H, T + 2)
    logits = torch.randn((T, E), generator=torch.Generator().manual_seed(T + 3)).to(dtype)
    w, ids = route(logits.float(), K)
    want, bound = O.experts(x.double().numpy(), w, ids, *weights)
    # float32 routing weights: exponentials, a sum of E terms and two divisions
    bound = bound + (E + 16) * 2.0 ** -23 * (np.abs(want) + bound)
    err = np.abs(_layer(x, logits, K, True, weights).double().cpu().numpy() - want)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("T", [65535, 70001])
def test_activations_past_32_bits(T):
    """x and out of just under and of more than 4 GiB: the last rows are those
    of a small call."""
    H, I, E = 32768, 128, 2
    weights = _weights(E, H, I, 15)
    dev = _dev(weights)
    ids, w = _routing(T, E, 1, 16)
    g = torch.Generator(device=DEV).manual_seed(17)
    x = torch.randn((T, H), generator=g, device=DEV, dtype=torch.bfloat16)
    got = _run(x, w, ids, dev)
    for part in (slice(0, 20), slice(T // 2, T // 2 + 20), slice(T - 20, T)):
        assert torch.equal(got[part], _run(x[part], w[part], ids[part], dev))
    part = slice(T - 3, T)
    _close(got[part], x[part].cpu(), w[part], ids[part], weights)


@pytest.mark.parametrize("T", [1, 40, 200])
def test_largest_expert(T):
    """An expert of nearly 2^31 values a matrix, all but its corners zero."""
    H, I = 32768, 65504
    rows, cols, outs = (0, 17, I - 18, I - 1), (0, 33, H - 32, H - 1), (0, 15, H - 16, H - 1)
    rng = np.random.default_rng(18)
    codes = [rng.integers(0, 16, (2, 4, 4)), rng.integers(0, 16, (4, 4))]
    w13 = torch.zeros((1, 2 * I, H // 2), dtype=torch.uint8, device=DEV)
    w2 = torch.zeros((1, H, I // 2), dtype=torch.uint8, device=DEV)
    s13 = torch.full((1, 2 * I, H // 32), 127, dtype=torch.uint8, device=DEV)
    s2 = torch.full((1, H, I // 32), 127, dtype=torch.uint8, device=DEV)
    # the same corners in an expert of 32 x 32, for the oracle
    small = [np.zeros((1, 64, 16), np.uint8), np.full((1, 64, 1), 127, np.uint8),
             np.zeros((1, 32, 16), np.uint8), np.full((1, 32, 1), 127, np.uint8)]

    def put(a, b, row, brow, col, bcol, code):
        a[0, row, col // 2] |= int(code) << (4 * (col % 2))
        b[0, brow, bcol // 2] |= int(code) << (4 * (bcol % 2))

    for i in range(4):
        for j in range(4):
            put(w13, small[0], rows[i], i, cols[j], j, codes[0][0, i, j])
            put(w13, small[0], I + rows[i], 32 + i, cols[j], j, codes[0][1, i, j])
            put(w2, small[2], outs[i], i, rows[j], j, codes[1][i, j])
    x = _x(T, H, 19)
    slots, w = np.zeros((T, 1), np.int32), np.full((T, 1), 0.75, np.float32)
    got = _run(x, w, slots, [w13, s13, w2, s2])
    assert int((got != 0).any(dim=0).sum()) <= 4
    xs = np.zeros((T, 32))
    xs[:, :4] = x.double().numpy()[:, list(cols)]
    want, bound = O.experts(xs, w, slots, *small)  # (what it leaves out adds exact zeros)
    assert np.abs(want[:, :4]).max() > 1
    err = np.abs(got[:, list(outs)].double().cpu().numpy() - want[:, :4])
    assert (err <= bound[:, :4]).all(), float((err / bound[:, :4]).max())


# ---------------------------------------------------------------------------
# Buffers as the C interface documents them
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("T,few", [(1, True), (12, True), (40, False)])
def test_act_and_work_of_the_documented_sizes(T, few):
    """Calls in buffers of exactly the documented bytes keep what stands behind
    them, and act itself where act stays in float32."""
    H, I, E, K = 96, 64, 5, 2
    weights = _weights(E, H, I, 20)
    dev = _dev(weights)
    ids, w = _routing(T, E, K, 21)
    x = _x(T, H, 22).to(DEV)
    tw, ts = torch.from_numpy(w).to(DEV), torch.from_numpy(ids).to(DEV)
    work_bytes = _lib.lib().wisp_moe_mxfp4_work_bytes(T, K, H, I, E)
    act_bytes = T * K * I * 2
    act = torch.full((act_bytes + 4096,), 7, dtype=torch.uint8, device=DEV)
    work = torch.full((work_bytes + 4096,), 7, dtype=torch.uint8, device=DEV)
    out = torch.full((T * H + 2048,), 7.0, dtype=torch.bfloat16, device=DEV)
    w13, s13, w2, s2 = dev
    _lib.check(_lib.lib().wisp_moe_experts_mxfp4(
        x.data_ptr(), T, H, I, K, tw.data_ptr(), ts.data_ptr(), E, w13.data_ptr(), w13.stride(0),
        s13.data_ptr(), s13.stride(0), w2.data_ptr(), w2.stride(0), s2.data_ptr(), s2.stride(0),
        act.data_ptr(), out.data_ptr(), work.data_ptr(), work_bytes, _lib.stream_handle()), "call")
    assert torch.equal(out[:T * H].view(T, H), _run(x, w, ids, dev))
    assert (act[act_bytes:] == 7).all() and (work[work_bytes:] == 7).all()
    assert (out[T * H:] == 7).all() and bool((act == 7).all()) == few


@pytest.mark.parametrize("T", [1, 30])
def test_a_layers_work_buffer_is_that_of_all_its_experts(T):
    """wisp_layer_forward in a work buffer of wisp_moe_mxfp4_work_bytes with
    nslots = num_experts; a call without one is refused before the pager's state
    changes."""
    H, I, E, K, cap = 128, 2304, 6, 2, 4
    g = torch.Generator().manual_seed(23)
    m = mx.quantize_masters_mxfp4((torch.randn((E, 2 * I, H), generator=g) * 0.05).bfloat16(),
                                  (torch.randn((E, H, I), generator=g) * 0.05).bfloat16(), DEV)
    st = mx.WispMoEStateMxfp4(*m, cap, "paged", DEV, 0)
    x, lg = _x(T, H, 24).to(DEV), torch.randn((T, E), generator=g).to(DEV)
    out = torch.empty_like(x)
    ws = st._ws.ensure(T, K, cap)
    need = _lib.lib().wisp_moe_mxfp4_work_bytes(T, K, H, I, E)
    assert ws.work_bytes >= need

    def call(nbytes):
        ws.work_bytes = nbytes
        return _lib.lib().wisp_layer_forward(st._handle, x.data_ptr(), lg.data_ptr(), _lib.WISP_F32,
                                             T, K, 1, out.data_ptr(), C.byref(ws),
                                             _lib.WISP_ALGO_AUTO, _lib.stream_handle())

    assert call(0) == _lib.WISP_ERR_INVALID and st.expert_to_slot == {}
    assert call(need) == _lib.WISP_OK
    w13, w2, s13, s2 = (t.contiguous().to(DEV) for t in m)
    assert torch.equal(out, mx.route_and_experts_mxfp4(x, lg, K, True, w13, w2, s13, s2))


@pytest.mark.parametrize("T", [1, 40, 400])
def test_weights_past_float32_are_infinite(T):
    """Codes of the highest scales whose value is 2^128 or more, on one expert
    and row: infinite there as they read back, whatever the activation."""
    H, I, E = 128, 128, 2
    dev = _dev(_weights(E, H, I, 25))
    dev[0][1, 5, :16], dev[1][1, 5, 0] = 0x11, 254  # 2^126: finite
    ids, w = _routing(T, E, 1, 26)
    ids[0], x = 1, (_x(T, H, 27).double() * 2.0 ** -100).to(torch.bfloat16)
    assert torch.isfinite(mx.dequantize_mxfp4(dev[0], dev[1], torch.float32)).all()
    assert torch.isfinite(_run(x, w, ids, dev)).all()
    dev[0][1, 5, 3] = 0x74  # 2 * 2^127 and 6 * 2^127
    assert torch.isinf(mx.dequantize_mxfp4(dev[0], dev[1], torch.float32)).sum() == 2
    got = _run(x, w, ids, dev)
    hit = torch.from_numpy((ids == 1).any(axis=1)).to(DEV)
    assert torch.isfinite(got[~hit]).all() and not torch.isfinite(got[hit]).all(dim=1).any()
