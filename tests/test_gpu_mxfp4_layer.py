"""The paging state over MXFP4 experts: pager decisions bit-exact with the
oracle, paged outputs byte-identical to resident ones and within the derived
bound of the oracle, on both page-in engines, over resizes and prefetches; and
the plug-in's quantisation of a bf16 layer."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as O
from oracle.moe import route
from oracle.pager import PagerOracle
from wisp.integrations.vllm import fused_moe as fm
from wisp.integrations.vllm import fused_moe_mxfp4 as mx
from wisp.integrations.vllm import layer as L
from wisp_amd import _lib

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
H, I, E, K = 288, 160, 12, 3


@pytest.fixture(scope="module")
def masters():
    g = torch.Generator().manual_seed(1)
    w13 = (torch.randn((E, 2 * I, H), generator=g) * 0.05).to(torch.bfloat16)
    w2 = (torch.randn((E, H, I), generator=g) * 0.05).to(torch.bfloat16)
    return mx.quantize_masters_mxfp4(w13, w2, DEV)


def _calls(tokens, seed, logits=torch.float32):
    g = torch.Generator().manual_seed(seed)
    for T in tokens:
        yield (torch.randn((T, H), generator=g).to(torch.bfloat16),
               torch.randn((T, E), generator=g).to(logits))


def _resident(masters):
    st = mx.WispMoEStateMxfp4(*masters, E, "resident", DEV, 1)
    st.prime_identity()
    return st


def _close(got, x, lg, masters):
    w, ids = route(lg.float(), K)
    want, bound = O.experts(x.double().numpy(), w, ids, masters[0].numpy(), masters[2].numpy(),
                            masters[1].numpy(), masters[3].numpy())
    bound = bound + (E + 16) * 2.0 ** -23 * (np.abs(want) + bound)  # float32 routing weights
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound).all(), float((err / bound).max())


def test_quantised_masters_are_one_slab(masters):
    lay = mx.Mxfp4SlabLayout(H, I)
    assert all(t.is_pinned() for t in masters)
    assert [t.data_ptr() - masters[0].data_ptr() for t in masters] == lay.offsets
    assert all(t.stride(0) == lay.slab for t in masters)
    assert lay.used == 3 * H * I * 17 // 32


@pytest.mark.parametrize("engine", ["kernel", "memcpy"])
@pytest.mark.parametrize("logits", [torch.float32, torch.bfloat16])
def test_paged_trace(masters, monkeypatch, engine, logits):
    """Calls of one token, of a few, of several groups, and none."""
    monkeypatch.setenv("WISP_PAGEIN_ENGINE", engine)
    st = mx.WispMoEStateMxfp4(*masters, 5, "paged", DEV, 0)
    assert st.pagein_engine == engine
    res, ora = _resident(masters), PagerOracle(E, 5)
    tokens = [1] * 8 + [2, 1, 4, 7, 1, 0, 13, 30, 1, 90, 3]
    for n, (x, lg) in enumerate(_calls(tokens, 2, logits)):
        got = st.forward(x.to(DEV), lg.to(DEV), K, True)
        ref = res.forward(x.to(DEV), lg.to(DEV), K, True)
        if len(x):
            ora.forward(route(lg.float(), K)[1].tolist())
        torch.cuda.synchronize()
        assert torch.equal(got, ref), n
        assert st.slot_to_expert == ora.slot_to_expert, n
        if n % 4 == 0 and len(x):
            _close(got, x, lg, masters)
    assert (st.stats_miss, st.stats_evict) == (ora.stats_miss, ora.stats_evict)
    assert res.stats_forward == len(tokens)


@pytest.mark.parametrize("H,I,tokens", [(256, 256, [1, 400, 30, 700]), (128, 2304, [5, 20, 60, 1]),
                                        (128, 12800, [40, 350])])
def test_paged_equals_resident(H, I, tokens):
    """Where a resident call runs in block tiles or w2's k range in parts."""
    E, K, g = 6, 2, torch.Generator().manual_seed(11)
    w13 = (torch.randn((E, 2 * I, H), generator=g) * 0.05).to(torch.bfloat16)
    w2 = (torch.randn((E, H, I), generator=g) * 0.05).to(torch.bfloat16)
    m = mx.quantize_masters_mxfp4(w13, w2, DEV)
    st = mx.WispMoEStateMxfp4(*m, 3, "paged", DEV, 0)
    res = mx.WispMoEStateMxfp4(*m, E, "resident", DEV, 1)
    res.prime_identity()
    dev = [t.contiguous().to(DEV) for t in m]
    for T in tokens:
        x = torch.randn((T, H), generator=g).to(torch.bfloat16).to(DEV)
        lg = torch.randn((T, E), generator=g).to(DEV)
        got = st.forward(x, lg, K, True)
        assert torch.equal(got, res.forward(x, lg, K, True)), T
        assert torch.equal(got, mx.route_and_experts_mxfp4(x, lg, K, True, *dev)), T


def test_slots_hold_the_masters_bytes(masters):
    st = mx.WispMoEStateMxfp4(*masters, 5, "paged", DEV, 0)
    for x, lg in _calls([1, 2, 9], 3):
        st.forward(x.to(DEV), lg.to(DEV), K, True)
    torch.cuda.synchronize()
    for e, s in st.expert_to_slot.items():
        for part in ("w13", "w2", "s13", "s2"):
            assert torch.equal(getattr(st, "scratch_" + part)[s].cpu(),
                               getattr(st, "cpu_" + part)[e]), (e, part)


def test_separate_masters(masters):
    """Masters that are not views of one slab, pinned or pageable."""
    res = _resident(masters)
    calls = list(_calls([1, 3, 8], 4))
    for pin in (True, False):
        own = [t.contiguous().clone() for t in masters]
        own = [t.pin_memory() if pin else t for t in own]
        st = mx.WispMoEStateMxfp4(*own, 4, "paged", DEV, 0)
        assert st.pagein_engine == ("kernel" if pin else "memcpy")
        for x, lg in calls:
            assert torch.equal(st.forward(x.to(DEV), lg.to(DEV), K, True),
                               res.forward(x.to(DEV), lg.to(DEV), K, True))


def test_resize(masters):
    st, res, ora = mx.WispMoEStateMxfp4(*masters, 4, "paged", DEV, 0), _resident(masters), \
        PagerOracle(E, 4)
    plan = {3: 7, 6: 3, 9: 99, 12: 5}
    for n, (x, lg) in enumerate(_calls([1, 2] * 8, 5)):
        if n in plan:
            torch.cuda.synchronize()
            st.resize_cap(plan[n])
            ora.resize_cap(plan[n])
        got = st.forward(x.to(DEV), lg.to(DEV), K, True)
        ora.forward(route(lg, K)[1].tolist())
        assert torch.equal(got, res.forward(x.to(DEV), lg.to(DEV), K, True)), n
        torch.cuda.synchronize()
        assert st.slot_to_expert == ora.slot_to_expert, n


def test_prefetch(masters):
    st, res = mx.WispMoEStateMxfp4(*masters, 6, "paged", DEV, 0), _resident(masters)
    for n, (x, lg) in enumerate(_calls([1] * 6, 6)):
        st.prefetch_async([int(e) for e in route(lg, K)[1][0]])
        miss = st.stats_miss
        got = st.forward(x.to(DEV), lg.to(DEV), K, True)
        torch.cuda.synchronize()
        assert torch.equal(got, res.forward(x.to(DEV), lg.to(DEV), K, True))
        if n:
            assert st.stats_miss == miss  # what was predicted had been loaded


def test_two_layers_and_streams(masters):
    """Two states over the same masters on two streams at once."""
    a, b, res = mx.WispMoEStateMxfp4(*masters, 4, "paged", DEV, 0), \
        mx.WispMoEStateMxfp4(*masters, 5, "paged", DEV, 1), _resident(masters)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for x, lg in _calls([1, 4, 20], 7):
        x, lg = x.to(DEV), lg.to(DEV)
        want = res.forward(x, lg, K, True)
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            u = a.forward(x, lg, K, True)
        with torch.cuda.stream(s2):
            v = b.forward(x, lg, K, True)
        torch.cuda.synchronize()
        assert torch.equal(u, want) and torch.equal(v, want)


def test_timing_counts_the_calls(masters):
    st = _resident(masters)
    st.profile(True)
    for x, lg in _calls([1, 40], 8):
        st.forward(x.to(DEV), lg.to(DEV), K, True)
    torch.cuda.synchronize()
    p = st.profile(False)
    assert p["calls"] == 2 and p["w13_calls"] == 2 and p["w13"] > 0 and p["w2"] > 0


def test_state_refusals(masters):
    w13, w2, s13, s2 = masters
    ok = [w13, w2, s13, s2]
    for i, bad in ((0, w13.to(DEV)), (0, w13.float()), (1, w2[:, :, :16]), (2, s13[:3]),
                   (3, s2.transpose(1, 2).contiguous().transpose(1, 2)), (0, w13[0])):
        with pytest.raises(ValueError):
            mx.WispMoEStateMxfp4(*(ok[:i] + [bad] + ok[i + 1:]), 4, "paged", DEV, 0)
    for cap in (0, E + 1):
        with pytest.raises(ValueError):
            mx.WispMoEStateMxfp4(*ok, cap, "paged", DEV, 0)
    st = mx.WispMoEStateMxfp4(*ok, 2, "paged", DEV, 0)
    x, lg = next(_calls([1], 9))
    with pytest.raises(_lib.SubBatchError):  # one token needs more experts than there are slots
        st.forward(x.to(DEV), lg.to(DEV), K, True)
    st = mx.WispMoEStateMxfp4(*ok, 4, "paged", DEV, 0)
    with pytest.raises(ValueError):
        st.forward(x.float().to(DEV), lg.to(DEV), K, True)
    with pytest.raises(NotImplementedError):
        st.forward(x.to(DEV), lg.to(DEV), K, True, algo=_lib.WISP_ALGO_MFMA)
    with pytest.raises(ValueError):
        mx.Mxfp4SlabLayout(48, 64)
    with pytest.raises(ValueError):
        mx.quantize_masters_mxfp4(torch.zeros((2, 64, 64)), torch.zeros((2, 64, 64)), DEV)


# ---------------------------------------------------------------------------
# The plug-in
# ---------------------------------------------------------------------------


@pytest.fixture
def patched(monkeypatch):
    cls = L.UnquantizedFusedMoEMethod
    orig = (cls.create_weights, cls.process_weights_after_loading, cls.forward_cuda)
    monkeypatch.setenv("WISP_EXPERT_FORMAT", "mxfp4")
    yield
    cls.create_weights, cls.process_weights_after_loading, cls.forward_cuda = orig
    if hasattr(cls, "_wisp_patched"):
        delattr(cls, "_wisp_patched")
    fm._LAYER_STATES.clear()
    fm._LAYER_BY_ID.clear()


def _layer(dtype=torch.bfloat16, h=H, i=I):
    g = torch.Generator().manual_seed(10)
    m = L.FusedMoE(E, K, h, i, dtype)
    w13 = (torch.randn((E, 2 * i, h), generator=g) * 0.05).to(dtype)
    w2 = (torch.randn((E, h, i), generator=g) * 0.05).to(dtype)
    m.load_weights(w13, w2)
    m.process_weights_after_loading()
    return m, w13, w2


@pytest.mark.parametrize("mode", ["paged", "resident"])
def test_plugin_quantises_a_layer(patched, mode):
    fm.install_wisp_moe(mode=mode, cap_experts=4)
    m, w13, w2 = _layer()
    st = m._wisp_state
    assert isinstance(st, mx.WispMoEStateMxfp4) and fm._LAYER_STATES == [st]
    assert st.cap_experts == (4 if mode == "paged" else E) and m.w13_weight.numel() == 0
    assert fm.expert_bytes_per_cap() == 3 * H * I * 17 // 32
    (q13, s13), (q2, s2) = mx.quantize_mxfp4(w13.to(DEV)), mx.quantize_mxfp4(w2.to(DEV))
    for x, lg in _calls([1, 3, 40], 11):
        x, lg = x.to(DEV), lg.to(DEV)
        assert torch.equal(m(x, lg), mx.route_and_experts_mxfp4(x, lg, K, True, q13, q2, s13, s2))
    if mode == "paged":
        assert fm.resize_layer_caps(6) == 1 and st.cap_experts == 6


def test_plugin_refusals(patched):
    fm.install_wisp_moe(mode="paged", cap_experts=4)
    with pytest.raises(NotImplementedError):
        _layer(torch.float32)
    with pytest.raises(ValueError):
        _layer(h=H + 16)
    fm.install_wisp_moe(mode="copy")
    with pytest.raises(NotImplementedError):
        _layer()
