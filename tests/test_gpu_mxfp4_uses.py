"""MXFP4 calls as programs make them besides the plain one: in place, captured
through a state, on the memcpy engine's side streams, behind the cross-layer
prefetch, from weights that were loaded on the GPU, with the most pairs of the
two launches and with NaN logits."""
import random

import numpy as np
import pytest
import torch

from oracle import mxfp4 as O
from oracle.cooccur import CooccurOracle, prefetch_glue
from oracle.moe import route
from oracle.pager import PagerOracle
from tests.test_gpu_mxfp4 import _close, _dev, _layer, _routing, _run, _weights, _x
from wisp.integrations.vllm import fused_moe as fm
from wisp.integrations.vllm import fused_moe_mxfp4 as mx
from wisp.integrations.vllm import layer as L

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("T,H,I,E,K", [(1, 512, 256, 16, 2), (40, 160, 96, 6, 2),
                                       (30, 128, 2304, 4, 2), (330, 256, 512, 4, 1)])
def test_out_may_be_x(T, H, I, E, K):
    dev = _dev(_weights(E, H, I, 1))
    ids, w = _routing(T, E, K, 2)
    x = _x(T, H, 3).to(DEV)
    want = _run(x, w, ids, dev)
    assert torch.equal(_run(x, w, ids, dev, out=x), want) and torch.equal(x, want)


@pytest.mark.parametrize("T,H,I,E,K", [(2, 64, 32, 70, 64), (8, 96, 64, 40, 16), (12, 64, 32, 8, 1)])
def test_most_pairs_of_the_two_launches(T, H, I, E, K):
    weights = _weights(E, H, I, 4)
    ids, w = _routing(T, E, K, 5)
    x = _x(T, H, 6)
    _close(_run(x, w, ids, weights), x, w, ids, weights)
    slots = ids.copy()
    slots[:, ::2] = -1
    _close(_run(x, w, slots, weights), x, w, slots, weights)


@pytest.mark.parametrize("T", [1, 40])
def test_nan_logits_rank_last(T):
    """They count as lowest: a token with enough others is routed as if they
    were -inf; a token of NaNs alone takes the lowest ids, with NaN weights."""
    E, H, I, K = 20, 64, 32, 4
    dev = _dev(_weights(E, H, I, 7))
    x = _x(T, H, 8)
    lg = torch.randn((T, E), generator=torch.Generator().manual_seed(9))
    low = lg.clone()
    lg[:, ::3], low[:, ::3] = float("nan"), float("-inf")
    assert torch.equal(_layer(x, lg, K, True, dev), _layer(x, low, K, True, dev))
    lg[0] = float("nan")
    got = _layer(x, lg, K, True, dev)
    assert torch.isnan(got[0]).all()
    assert torch.equal(got[1:], _layer(x, low, K, True, dev)[1:])


def _masters(E, H, I, seed):
    g = torch.Generator().manual_seed(seed)
    w13 = (torch.randn((E, 2 * I, H), generator=g) * 0.05).to(torch.bfloat16)
    w2 = (torch.randn((E, H, I), generator=g) * 0.05).to(torch.bfloat16)
    return w13, w2


def _resident(m, E):
    st = mx.WispMoEStateMxfp4(*m, E, "resident", DEV, 0)
    st.prime_identity()
    return st


@pytest.mark.parametrize("H,I", [(160, 96), (128, 2304), (256, 256)])
def test_resident_state_in_graphs(H, I):
    """Captured at three sizes on one state whose buffers hold the largest,
    replayed in turn with eager calls between."""
    E, K = 6, 2
    st = _resident(mx.quantize_masters_mxfp4(*_masters(E, H, I, 10), DEV), E)
    sets = []
    for T in (400, 30, 1):
        x, lg = _x(T, H, T).to(DEV), torch.randn((T, E), device=DEV)
        out = torch.empty_like(x)
        st.forward(x, lg, K, True, out=out)
        sets.append((x, lg, out))
    graphs = []
    for x, lg, out in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            st.forward(x, lg, K, True, out=out)
        graphs.append(g)
    for _ in range(3):
        want = []
        for x, lg, out in sets:
            x.mul_(-0.5)
            lg.copy_(lg.flip(1))
            want.append(st.forward(x, lg, K, True))
            out.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, _, out), b in zip(sets, want):
            assert torch.equal(out, b)


@pytest.mark.parametrize("streams", ["1", "2"])
@pytest.mark.parametrize("cap", [4, 9])
def test_memcpy_engine_on_side_streams(monkeypatch, streams, cap):
    E, H, I, K = 12, 160, 96, 3
    monkeypatch.setenv("WISP_PAGEIN_ENGINE", "memcpy")
    monkeypatch.setenv("WISP_PAGEIN_STREAMS", streams)
    m = mx.quantize_masters_mxfp4(*_masters(E, H, I, 11), DEV)
    st, res, ora = mx.WispMoEStateMxfp4(*m, cap, "paged", DEV, 0), _resident(m, E), \
        PagerOracle(E, cap)
    g = torch.Generator().manual_seed(12)
    for T in [1] * 6 + [2, 30, 1, 3, 90, 1]:
        x = torch.randn((T, H), generator=g).to(torch.bfloat16).to(DEV)
        lg = torch.randn((T, E), generator=g)
        got, want = st.forward(x, lg.to(DEV), K, True), res.forward(x, lg.to(DEV), K, True)
        ora.forward(route(lg, K)[1].tolist())
        torch.cuda.synchronize()
        assert torch.equal(got, want) and st.slot_to_expert == ora.slot_to_expert, T


def test_cross_layer_prefetch(monkeypatch):
    """A stack of MXFP4 layers with the online co-occurrence table: decisions
    as the oracle's, outputs as the resident layer's."""
    layers, cap, E, H, I, K = 4, 4, 16, 64, 32, 2
    m = mx.quantize_masters_mxfp4(*_masters(E, H, I, 13), DEV)
    monkeypatch.setenv("WISP_COOCCUR_ONLINE", "1")
    monkeypatch.delenv("WISP_COOCCUR_PATH", raising=False)
    monkeypatch.setenv("WISP_PREFETCH", "1")
    fm._reset_cooccur()
    states = [mx.WispMoEStateMxfp4(*m, cap, "paged", DEV, n) for n in range(layers)]
    monkeypatch.setattr(fm, "_LAYER_STATES", states)
    res, table, obs = _resident(m, E), CooccurOracle(), {}
    oras = [PagerOracle(E, cap) for _ in range(layers)]
    rng = random.Random(14)
    x = _x(1, H, 15).to(DEV)
    try:
        for step in range(24):
            for n in range(layers):
                lg = torch.tensor([rng.sample(range(E), E)], dtype=torch.float32)
                lg[0, (3 * n + step % 3) % E] += 20
                got = states[n].forward(x, lg.to(DEV), K, True)
                fm._prefetch_after_forward(states[n])
                want = res.forward(x, lg.to(DEV), K, True)
                oras[n].forward(route(lg, K)[1].tolist())
                prefetch_glue(oras, n, table, obs, online=True)
                torch.cuda.synchronize()
                assert torch.equal(got, want), (step, n)
            for s, o in zip(states, oras):
                assert s.slot_to_expert == o.slot_to_expert and s.lru_tick == o.lru_tick
                assert (s.stats_miss, s.stats_pred_total) == (o.stats_miss, o.stats_pred_total)
        assert sum(o.stats_pred_total for o in oras) > 0
    finally:
        fm._reset_cooccur()


@pytest.mark.parametrize("where", ["cuda:0", "cpu"])
def test_plugin_on_weights_loaded_elsewhere(monkeypatch, where):
    """The method was patched after the layer had made its weights."""
    E, H, I, K = 6, 160, 96, 2
    cls = L.UnquantizedFusedMoEMethod
    orig = (cls.create_weights, cls.process_weights_after_loading, cls.forward_cuda)
    monkeypatch.setenv("WISP_EXPERT_FORMAT", "mxfp4")
    w13, w2 = _masters(E, H, I, 16)
    m = L.FusedMoE(E, K, H, I)
    m.w13_weight.data, m.w2_weight.data = w13.to(where), w2.to(where)
    try:
        fm.install_wisp_moe(mode="paged", cap_experts=3)
        m.process_weights_after_loading()
        m.process_weights_after_loading()  # once is enough
        assert len(fm._LAYER_STATES) == 1 and m.w13_weight.numel() == 0
        (q13, s13), (q2, s2) = (mx.quantize_mxfp4(w.to(DEV)) for w in (w13, w2))
        for T in (1, 25):
            x = _x(T, H, T).to(DEV)
            lg = torch.randn((T, E), generator=torch.Generator().manual_seed(T)).to(DEV)
            assert torch.equal(m(x, lg), mx.route_and_experts_mxfp4(x, lg, K, True, q13, q2, s13,
                                                                    s2))
    finally:
        cls.create_weights, cls.process_weights_after_loading, cls.forward_cuda = orig
        if hasattr(cls, "_wisp_patched"):
            delattr(cls, "_wisp_patched")
        fm._LAYER_STATES.clear()
        fm._LAYER_BY_ID.clear()


@pytest.mark.parametrize("T,H,I,E,K", [(2, 64, 32, 600, 3), (300, 64, 32, 600, 3)])
def test_two_streams_at_once(T, H, I, E, K):
    """The same weights and inputs on two streams whose work overlaps."""
    weights = _weights(E, H, I, 17)
    dev = _dev(weights)
    ids, w = _routing(T, E, K, 18)
    xs = [_x(T, H, 19).to(DEV), _x(T, H, 20).to(DEV)]
    tw, ts = torch.from_numpy(w).to(DEV), torch.from_numpy(np.asarray(ids)).to(DEV)
    w13, s13, w2, s2 = dev
    want = [mx.experts_mxfp4(x, tw, ts, w13, w2, s13, s2) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(mx.experts_mxfp4(xs[i], tw, ts, w13, w2, s13, s2))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    bound = O.experts(xs[0].double().cpu().numpy(), w, ids, *weights)
    assert (np.abs(want[0].double().cpu().numpy() - bound[0]) <= bound[1]).all()
