"""Grouped products on the GPU against the float64 oracle: within what a
float32 sum and one rounding allow (derived in ``oracle.rows.grouped_mm``), at
sizes, groups, strides and values where they can go wrong."""
import numpy as np
import pytest
import torch

from oracle import rows as O
from wisp.integrations.vllm import grouped_mm as G
from wisp.integrations.vllm import rows_fp8 as R
from wisp_amd import _lib

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn

# The fp8 matrix instruction aligns the products of a block of 128 to its largest
# one before it sums them and keeps at least 12 bits behind the point there:
# measured, up to 1.7e-4 of the sum of the products' sizes on codes of the full
# range, 1.3e-5 on quantised normal values.
DOT8 = 2.0 ** -12


def _f64(t):
    return t.detach().cpu().double().numpy()


def _bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def _randn(shape, seed, dtype=BF, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _ends(counts):
    return torch.tensor(np.cumsum(counts), dtype=torch.int32, device=DEV)


def _near(got, want, bound, dtype):
    half = O.BF16 if dtype == BF else O.STEP
    bound = bound + half * (np.abs(want) + bound) + O.TINY
    d = np.abs(_f64(got) - want)
    assert got.dtype == dtype
    assert np.all(d <= bound), float((d / bound).max())


def _fp8(v):
    """Codes of any values (to the nearest), by torch's cast."""
    return v.clamp(-448, 448).to(FP8)


def _case8(M, E, N, K, seed):
    """Rows and weights in FP8 as they are made, scales of unequal size."""
    q = _fp8(_randn((M, K), seed, F32, 100.0))
    w = _fp8(_randn((E, N, K), seed + 1, F32, 100.0))
    g, b = -(-K // 128), -(-N // 128)
    s = torch.exp(_randn((M, g), seed + 2, F32)) * 0.01
    ws = torch.exp(_randn((E, b, g), seed + 3, F32)) * 0.001
    return q, s, w, ws


def _values8(q, s, w, ws):
    K, N = q.shape[1], w.shape[1]
    x = _f64(q.float()) * np.repeat(_f64(s), 128, axis=1)[:, :K]
    return x, _f64(w.float()) * O.spread(_f64(ws), N, K)


def _check(M, E, N, K, counts, seed=0, dtype=BF):
    x, w = _randn((M, K), seed), _randn((E, N, K), seed + 1, BF, 0.1)
    ends = _ends(counts)
    got = G.grouped_mm(x, w, ends, dtype=dtype)
    _near(got, *O.grouped_mm(_f64(x), _f64(w), ends.tolist()), dtype)
    return got


def _check8(M, E, N, K, counts, seed=0):
    case = _case8(M, E, N, K, seed)
    ends = _ends(counts)
    got = G.grouped_mm_fp8(*case, ends)
    _near(got, *O.grouped_mm(*_values8(*case), ends.tolist(), DOT8), BF)
    return got


def _spread_counts(M, E, seed):
    """Ragged counts with empty groups."""
    r = np.random.RandomState(seed)
    p = r.exponential(size=E) * (r.rand(E) < 0.7)
    p = p if p.sum() else np.ones(E)
    return r.multinomial(M, p / p.sum())


# rows, experts, outputs, columns
SIZES = [(1, 1, 1, 16), (1, 4, 8, 16), (5, 3, 17, 32), (16, 2, 64, 64), (17, 1, 100, 80),
         (33, 5, 256, 128), (64, 1, 257, 144), (65, 2, 130, 272), (100, 7, 300, 352),
         (231, 24, 704, 1056), (130, 1, 512, 256), (300, 2, 264, 512), (515, 3, 128, 176),
         (1000, 4, 192, 1040), (600, 1, 320, 2048), (9, 130, 48, 64), (1100, 300, 40, 48)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,E,N,K", SIZES)
def test_bf16_sizes(M, E, N, K, dtype):
    _check(M, E, N, K, _spread_counts(M, E, M + N), M + K, dtype)


@pytest.mark.parametrize("M,E,N,K", SIZES)
def test_fp8_sizes(M, E, N, K):
    _check8(M, E, N, K, _spread_counts(M, E, M + N), M + K)


@pytest.mark.parametrize("K", [8, 24, 56, 72, 120, 136, 184, 200, 1000])
def test_bf16_columns(K):
    _check(40, 3, 70, K, [13, 0, 27], K)


@pytest.mark.parametrize("K", [16, 48, 112, 128, 144, 240, 256, 272, 400, 1008])
def test_fp8_columns(K):
    _check8(40, 3, 150, K, [13, 0, 27], K)


COUNTS = [[0, 0, 0], [0, 0, 1], [1, 0, 0], [64, 64, 64], [63, 65, 1], [128, 0, 129], [300, 1, 15],
          [16, 17, 256], [257, 255, 3], [0, 700, 0], [1, 1, 1]]


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("tail", [0, 1, 37])
def test_groups(counts, tail):
    """Groups around the tiles' sizes, empty ones, and rows behind the last."""
    M = sum(counts) + tail
    if M:
        _check(M, 3, 72, 96, counts, M)
        _check8(M, 3, 72, 96, counts, M)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 8, 15, 16, 17, 40, 64, 70, 128, 140, 256, 300])
def test_rows_do_not_depend_on_their_group_s_size(rows, fp8):
    """A group's rows and the same rows one by one agree within the bound."""
    if fp8:
        _check8(rows, 1, 96, 256, [rows], rows)
    else:
        _check(rows, 1, 96, 256, [rows], rows)


@pytest.mark.parametrize("fp8", [False, True])
def test_ends_that_descend_or_lie_outside(fp8):
    M, E, N, K = 90, 6, 40, 64
    for ends in ([10, 5, 30, 200, 100, 95], [-3, -1, 50, 20, 60, 60], [0, 0, 0, 0, 0, 0],
                 [2 ** 31 - 1] * 6, [-2 ** 31] * 6, [90, 0, 0, 0, 0, 0]):
        e = torch.tensor(ends, dtype=torch.int32, device=DEV)
        if fp8:
            case = _case8(M, E, N, K, 3)
            _near(G.grouped_mm_fp8(*case, e), *O.grouped_mm(*_values8(*case), ends, DOT8), BF)
        else:
            x, w = _randn((M, K), 1), _randn((E, N, K), 2)
            _near(G.grouped_mm(x, w, e), *O.grouped_mm(_f64(x), _f64(w), ends), BF)


@pytest.mark.parametrize("N", [64, 41])
def test_rows_behind_the_last_group(N):
    """Left as they are in a given output, zero in a new one."""
    x, w = _randn((200, 64), 4), _randn((3, N, 64), 5)
    for counts in ([20, 0, 33], [0, 0, 0], [100, 50, 50], [100, 50, 49]):
        n, ends = sum(counts), _ends(counts)
        for dtype in (BF, F32):
            new = G.grouped_mm(x, w, ends, dtype=dtype)
            assert not new[n:].any() and not torch.isnan(new).any()
            out = torch.full((200, N), float("nan"), dtype=dtype, device=DEV)
            assert G.grouped_mm(x, w, ends, dtype=dtype, out=out) is out
            assert torch.equal(out[:n], new[:n]) and out[n:].isnan().all()
    case = _case8(200, 3, N, 64, 6)
    out = torch.full((200, N), float("nan"), dtype=BF, device=DEV)
    G.grouped_mm_fp8(*case, ends, out=out)
    new = G.grouped_mm_fp8(*case, ends)
    assert torch.equal(out[:199], new[:199]) and out[199].isnan().all() and not new[199].any()


def test_values_stay_in_their_rows_and_columns():
    """Infinities and NaNs in rows of another group, behind the last group, in
    another expert's weights, in the columns behind a row's end and in rows
    between the ones in use touch nothing else."""
    M, E, N, K = 70, 3, 80, 72
    big_x = torch.full((M, 128), float("nan"), dtype=BF, device=DEV)
    big_w = torch.full((E, N + 5, 96), float("nan"), dtype=BF, device=DEV)
    x, w = _randn((M, K), 7), _randn((E, N, K), 8)
    big_x[:, :K], big_w[:, :N, :K] = x, w
    ends = _ends([30, 0, 21])
    want = G.grouped_mm(x, w, ends)
    big_x[51:] = float("nan")
    big_w[1] = float("inf")
    assert torch.equal(G.grouped_mm(big_x[:, :K], big_w[:, :N, :K], ends), want)
    big_x[33, 9], big_w[0, 4, 11] = float("inf"), float("nan")
    got = G.grouped_mm(big_x[:, :K], big_w[:, :N, :K], ends)
    bad = torch.zeros((M, N), dtype=torch.bool, device=DEV)
    bad[33] = True
    bad[:30, 4] = True
    assert torch.equal(got[~bad], want[~bad]) and not torch.isfinite(got[bad]).any()


def test_fp8_values_stay_in_their_rows_and_columns():
    M, E, N, K = 70, 3, 150, 144
    q, s, w, ws = _case8(M, E, N, K, 9)
    big_q = torch.full((M, 256), 0x7f, dtype=torch.uint8, device=DEV).view(FP8)
    big_w = torch.full((E, N + 3, 192), 0x7f, dtype=torch.uint8, device=DEV).view(FP8)
    big_s = torch.full((M, 5), float("nan"), device=DEV)
    big_q.view(torch.uint8)[:, :K], big_w.view(torch.uint8)[:, :N, :K] = \
        q.view(torch.uint8), w.view(torch.uint8)
    big_s[:, :2] = s
    ends = _ends([30, 0, 21])
    want = G.grouped_mm_fp8(q, s, w, ws, ends)
    big_q.view(torch.uint8)[51:] = 0x7f
    big_s[51:] = float("inf")
    big_w.view(torch.uint8)[1] = 0x7f
    ws = ws.clone()
    ws[1] = float("nan")
    got = G.grouped_mm_fp8(big_q[:, :K], big_s[:, :2], big_w[:, :N, :K], ws, ends)
    assert torch.equal(got, want)
    big_s[33, 1] = float("inf")
    ws[0, 1, 0] = float("nan")
    got = G.grouped_mm_fp8(big_q[:, :K], big_s[:, :2], big_w[:, :N, :K], ws, ends)
    bad = torch.zeros((M, N), dtype=torch.bool, device=DEV)
    bad[33] = True
    bad[:30, 128:] = True
    assert torch.equal(got[~bad], want[~bad]) and not torch.isfinite(got[bad]).any()


@pytest.mark.parametrize("M", [30, 400])
def test_strides(M):
    """Rows and experts any distance apart, unaligned and transposed rows."""
    E, N, K = 3, 56, 136
    base, wide = _randn((M, 400), 10), _randn((E, N, 160), 11)
    ends = _ends([M // 3, M // 3, M // 4])
    w = wide[:, :, :K]
    want = G.grouped_mm(base[:, 40:40 + K].contiguous(), w.contiguous(), ends)
    assert torch.equal(G.grouped_mm(base[:, 40:40 + K], w, ends), want)
    slab = torch.empty(E, N * K + 24, dtype=BF, device=DEV)
    apart = slab[:, 8:8 + N * K].view(E, N, K)
    apart.copy_(w)
    assert torch.equal(G.grouped_mm(base[:, 40:40 + K], apart, ends), want)
    off = G.grouped_mm(base[:, 41:41 + K], w, ends)   # unaligned rows are copied
    assert torch.equal(off, G.grouped_mm(base[:, 41:41 + K].contiguous(), w, ends))
    t = base[:, :K].t().contiguous().t()
    assert torch.equal(G.grouped_mm(t, w, ends), G.grouped_mm(base[:, :K].contiguous(), w, ends))
    one = G.grouped_mm(base[:, :K], w[:1].expand(E, N, K), ends)   # experts that share weights
    assert torch.equal(one, G.grouped_mm(base[:, :K], w[:1].repeat(E, 1, 1), ends))
    K = 144
    q, s, w8, ws = _case8(M, E, N, K, 12)
    want = G.grouped_mm_fp8(q, s, w8, ws, ends)
    sw = torch.empty((M, 9), device=DEV)[:, 3:5].copy_(s)
    slab = torch.zeros((E, 4 * N * K), dtype=torch.uint8, device=DEV)
    apart = slab[:, 16:16 + N * K].view(E, N, K)
    apart.copy_(w8.view(torch.uint8))
    assert torch.equal(G.grouped_mm_fp8(q, sw, apart.view(FP8), ws, ends), want)
    assert torch.equal(G.grouped_mm_fp8(q, s.t().contiguous().t(), w8, ws, ends), want)


def test_expert_weights_beyond_32_bits():
    """An expert's place past 2^32 bytes."""
    E, N, K = 5, 16384, 32768
    w = torch.zeros((E, N, K), dtype=BF, device=DEV)
    w[4, -300:] = _randn((300, K), 13, BF, 0.05)
    x = _randn((20, K), 14)
    got = G.grouped_mm(x, w, _ends([3, 0, 2, 0, 15]), dtype=F32)
    assert not got[:5].any() and not got[:, :-300].any()
    want, bound = O.grouped_mm(_f64(x[5:]), _f64(w[4:, -300:]), [15])
    _near(got[5:, -300:], want, bound, F32)


def test_rows_beyond_32_bits():
    """Rows and outputs past 2^32 bytes."""
    M, N, K = 140000, 16384, 16384
    x = torch.zeros((M, K), dtype=BF, device=DEV)
    x[-70:] = _randn((70, K), 15)
    w = _randn((2, 64, K), 16, BF, 0.05)
    full = torch.zeros((2, N, K), dtype=BF, device=DEV)
    full[:, -64:] = w
    got = G.grouped_mm(x, full, _ends([M - 40, 40]))
    want, bound = O.grouped_mm(_f64(x[-70:]), _f64(w), [30, 70])
    _near(got[-70:, -64:], want, bound, BF)
    assert not got[-70:, :-64].any() and not got[M - 2000:M - 70].any() and not got[:300].any()


@pytest.mark.parametrize("fp8", [False, True])
def test_as_many_rows_as_are_counted(fp8):
    """2^31 - 1 rows, all but three of them one group's: tiles and rows are counted
    beyond 2^31.  (Values that every order of the sum gives exactly.)"""
    M, N, K = 2 ** 31 - 1, 8, 16 if fp8 else 8
    if torch.cuda.get_device_properties(0).total_memory < 120 * 2 ** 30:
        pytest.skip("needs 90 GB")
    kind = FP8 if fp8 else BF
    g = torch.Generator().manual_seed(17)
    block = torch.randint(-3, 4, (2 ** 24, K), generator=g).to(DEV).float()
    w = torch.randint(-3, 4, (3, N, K), generator=g).to(DEV).float()
    want = [(block @ w[e].t()).to(BF) for e in (0, 2)]
    x = torch.empty((M, K), dtype=kind, device=DEV)
    part = block.to(kind)
    for i in range(0, M, 2 ** 24):
        x[i:i + 2 ** 24] = part[:min(2 ** 24, M - i)]
    ends = torch.tensor([M - 3, 0, M - 1], dtype=torch.int32, device=DEV)
    if fp8:
        out = G.grouped_mm_fp8(x, torch.ones((M, 1), device=DEV), w.to(FP8),
                               torch.ones((3, 1, 1), device=DEV), ends)
    else:
        out = G.grouped_mm(x, w.to(BF), ends)
    del x
    for i in range(0, M, 2 ** 24):
        n = min(2 ** 24, M - 3 - i)
        assert torch.equal(out[i:i + n], want[0][:n]), i
    assert torch.equal(out[M - 3:M - 1], want[1][2 ** 24 - 4:2 ** 24 - 2])
    assert not out[M - 1].any()
    del out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M", [12, 200, 900])
def test_runs_together(M):
    """The operators as a rank uses them, against the oracle's own chain from
    the codes each of them made."""
    E, H, I = 4, 256, 160
    x, res = _randn((M, H), 20), _randn((M, H), 21, BF, 3.0)
    weight = (1 + 0.1 * _randn((H,), 22, F32)).to(BF)
    w13, w2 = (torch.empty(s, dtype=FP8, device=DEV) for s in ((E, 2 * I, H), (E, H, I)))
    s13 = torch.empty((E, 3, 2), device=DEV)
    s2 = torch.empty((E, 2, 2), device=DEV)
    for w, s, seed in ((w13, s13, 23), (w2, s2, 24)):
        w.copy_(_fp8(_randn(w.shape, seed, F32, 100.0)))
        s.copy_(torch.exp(0.3 * _randn(s.shape, seed + 5, F32)) * 2e-4)
    ends = _ends(_spread_counts(M, E, M))
    n = int(ends[-1])
    q, s, r = R.add_rms_norm_fp8(x, weight, 1e-6, res)
    h = G.grouped_mm_fp8(q, s, w13, s13, ends)
    _near(h, *O.grouped_mm(*_values8(q, s, w13, s13), ends.tolist(), DOT8), BF)
    a, sa = R.silu_mul_fp8(h)
    y = G.grouped_mm_fp8(a, sa, w2, s2, ends)
    _near(y, *O.grouped_mm(*_values8(a, sa, w2, s2), ends.tolist(), DOT8), BF)
    # the whole chain without any rounding: three times eight bits
    v = O.rms_norm(_f64((x.double() + res.double()).to(BF)), _f64(weight), 1e-6)
    f13 = _f64(w13.float()) * O.spread(_f64(s13), 2 * I, H)
    f2 = _f64(w2.float()) * O.spread(_f64(s2), H, I)
    want, _ = O.grouped_mm(O.silu_mul(O.grouped_mm(v, f13, ends.tolist())[0])[0], f2,
                           ends.tolist())
    off = np.linalg.norm(_f64(y)[:n] - want[:n]) / np.linalg.norm(want[:n])
    # a code is off by at most 2^-4 of its value, each product averages over its
    # 160 or 256 columns: the rows' errors add as squares, 2^-4 per quantisation
    # at the very most (relative to the norm), twice for gate and up
    assert off <= 4 * 2.0 ** -4


@pytest.mark.parametrize("fp8", [False, True])
def test_in_a_graph_and_on_streams(fp8):
    """Captured and replayed with other ends, rows and weights in the same
    buffers, beside eager calls and a second graph; on a side stream."""
    M, E, N, K = 300, 5, 200, 272
    ins = _case8(M, E, N, K, 30) if fp8 else (_randn((M, K), 31), _randn((E, N, K), 32))
    call = G.grouped_mm_fp8 if fp8 else G.grouped_mm
    sets = [_ends(_spread_counts(M - k, E, k)) for k in range(4)]
    ends = sets[0].clone()
    call(*ins, ends)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(*ins, ends))
        graphs.append(g)
    for e in sets:
        ends.copy_(e)
        want = call(*ins, e)
        for g, out in zip(graphs, outs):
            out.fill_(7)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = call(*ins, sets[1])
    b = call(*ins, sets[2])
    side.synchronize()
    assert torch.equal(a, call(*ins, sets[1])) and torch.equal(b, call(*ins, sets[2]))


@pytest.mark.parametrize("fp8", [False, True])
def test_the_same_bytes_again(fp8):
    M, E, N, K = 700, 6, 320, 400
    ins = _case8(M, E, N, K, 40) if fp8 else (_randn((M, K), 41), _randn((E, N, K), 42))
    call = G.grouped_mm_fp8 if fp8 else G.grouped_mm
    ends = _ends(_spread_counts(M, E, 43))
    first = call(*ins, ends)
    for _ in range(3):
        assert torch.equal(_bits(call(*ins, ends)), _bits(first))


# The variants beyond the smallest tiles.  Few rows: one wave's columns in one
# and in several batches, groups of more rows than a pass takes.
@pytest.mark.parametrize("M,E,N", [(1, 4, 40), (32, 3, 100), (64, 2, 129)])
@pytest.mark.parametrize("K", [496, 512, 528, 768, 1008, 1296, 1536, 1808, 2064, 4112])
def test_few_rows_by_columns(M, E, N, K):
    counts = _spread_counts(M, E, K) if M > 1 else [0, 1, 0, 0]
    _check(M, E, N, K, counts, K)
    _check8(M, E, N, K, counts, K)


# rows, experts, outputs: 128 and 256 weight rows a tile, whole and ragged
WIDE = [(70, 60, 1664), (300, 60, 1672), (1100, 60, 1660), (101, 100, 2048), (700, 110, 1800),
        (2000, 100, 1804), (90, 60, 1667), (333, 100, 1801)]


@pytest.mark.parametrize("K", [16, 136, 256, 464])
@pytest.mark.parametrize("M,E,N", WIDE)
def test_wide_panels(M, E, N, K):
    counts = _spread_counts(M - 3, E, M + K)
    for dtype in (BF, F32):
        _check(M, E, N, K, counts, M, dtype)
    _check8(M, E, N, K - K % 16, counts, M)


# rows per expert, outputs, columns: of 24 experts, enough to fill the GPU with
# the large tiles.  Columns: one chunk and less, whole pairs of chunks, an odd
# number of chunks, a piece more.
LARGE = [(60, 2048, 128), (60, 1800, 176), (61, 1796, 64), (90, 1800, 256), (95, 2048, 144),
         (100, 1928, 16), (125, 2048, 384), (130, 1800, 1040), (131, 1800, 512), (190, 2040, 272),
         (200, 1808, 400)]


@pytest.mark.parametrize("kind", ["even", "ragged", "one", "edges"])
@pytest.mark.parametrize("per,N,K", LARGE)
def test_large_tiles(per, N, K, kind):
    E = 24
    M = E * per
    if kind == "even":
        counts = [per] * E
    elif kind == "one":
        counts = [0] * 5 + [M - 9] + [0] * 18
    elif kind == "edges":   # around the tiles' heights, as many as there is room for
        counts, left = [], M
        for n in ([255, 0, 257, 1, 192, 193, 127, 129, 16, 17, 0, 31] * 2):
            counts.append(min(n, left))
            left -= counts[-1]
    else:
        counts = _spread_counts(M - 70, E, per)
    if N % 8 == 0:
        _check(M, E, N, K, counts, per)
        _check8(M, E, N, K, counts, per)
    _check(M, E, N, K, counts, per, F32)


@pytest.mark.parametrize("E,per,N", [(6, 200, 2056), (6, 400, 2056), (3, 900, 2056),
                                     (9, 330, 1800), (20, 260, 2048), (40, 130, 1544)])
@pytest.mark.parametrize("K", [136, 256])
def test_large_tiles_that_do_not_fill_the_gpu(E, per, N, K):
    """Tiles for a part of the GPU, and for one turn of it and a part."""
    for counts in ([per] * E, _spread_counts(E * per - 5, E, per)):
        _check(E * per, E, N, K, counts, K)
        _check8(E * per, E, N, K - K % 16, counts, K)


@pytest.mark.parametrize("per", [60, 130])
def test_large_tiles_values_stay_in_their_rows_and_columns(per):
    """As above: other groups' rows, rows behind the last group, other experts'
    weights, columns behind a row's end."""
    E, N, K = 24, 1800, 200
    M = E * per
    counts = _spread_counts(M - 33, E, per)
    counts[3], counts[4] = counts[3] + counts[4], 0
    ends = _ends(counts)
    x, w = _randn((M, K), per), _randn((E, N, K), per + 1)
    want = G.grouped_mm(x, w, ends)
    big_x = torch.full((M, 264), float("nan"), dtype=BF, device=DEV)
    big_w = torch.full((E, N + 3, 328), float("nan"), dtype=BF, device=DEV)
    big_x[:, :K], big_w[:, :N, :K] = x, w
    big_x[M - 33:] = float("inf")
    big_w[4] = float("nan")
    xs, ws = big_x[:, :K], big_w[:, :N, :K]
    assert torch.equal(G.grouped_mm(xs, ws, ends), want)
    out = torch.full((M, N), 7.0, dtype=BF, device=DEV)
    G.grouped_mm(xs, ws, ends, out=out)
    assert torch.equal(out[:M - 33], want[:M - 33]) and bool((out[M - 33:] == 7).all())
    e = int(np.argmax(counts))
    first, n = int(sum(counts[:e])), int(counts[e])
    big_x[first + n // 2, 9], big_w[e, 1799, 199] = float("inf"), float("nan")
    got = G.grouped_mm(xs, ws, ends)
    bad = torch.zeros((M, N), dtype=torch.bool, device=DEV)
    bad[first + n // 2] = True
    bad[first:first + n, 1799] = True
    assert torch.equal(got[~bad], want[~bad]) and not torch.isfinite(got[bad]).any()


@pytest.mark.parametrize("K", [144, 400])
def test_large_fp8_tiles_values_stay_in_their_rows_and_columns(K):
    E, N, per = 24, 1800, 100
    M = E * per
    counts = _spread_counts(M - 33, E, K)
    counts[3], counts[4] = counts[3] + counts[4], 0
    ends = _ends(counts)
    q, s, w, ws = _case8(M, E, N, K, K)
    g = s.shape[1]
    want = G.grouped_mm_fp8(q, s, w, ws, ends)
    big_q = torch.full((M, 528), 0x7f, dtype=torch.uint8, device=DEV).view(FP8)
    big_w = torch.full((E, N + 3, 448), 0x7f, dtype=torch.uint8, device=DEV).view(FP8)
    big_s = torch.full((M, g + 2), float("nan"), device=DEV)
    big_q.view(torch.uint8)[:, :K], big_w.view(torch.uint8)[:, :N, :K] = \
        q.view(torch.uint8), w.view(torch.uint8)
    big_s[:, :g] = s
    big_q.view(torch.uint8)[M - 33:] = 0x7f
    big_s[M - 33:] = float("inf")
    big_w.view(torch.uint8)[4] = 0x7f
    ws = ws.clone()
    ws[4] = float("nan")
    args = big_q[:, :K], big_s[:, :g], big_w[:, :N, :K], ws, ends
    assert torch.equal(G.grouped_mm_fp8(*args), want)
    out = torch.full((M, N), 7.0, dtype=BF, device=DEV)
    G.grouped_mm_fp8(*args, out=out)
    assert torch.equal(out[:M - 33], want[:M - 33]) and bool((out[M - 33:] == 7).all())
    e = int(np.argmax(counts))
    first, n = int(sum(counts[:e])), int(counts[e])
    big_s[first + n // 2, g - 1], ws[e, 14, 0] = float("inf"), float("nan")
    got = G.grouped_mm_fp8(*args)
    bad = torch.zeros((M, N), dtype=torch.bool, device=DEV)
    bad[first + n // 2] = True
    bad[first:first + n, 14 * 128:] = True
    assert torch.equal(got[~bad], want[~bad]) and not torch.isfinite(got[bad]).any()


@pytest.mark.parametrize("M,E,N", [(12, 3, 300), (90, 3, 300), (2400, 24, 1800), (4800, 24, 1800)])
@pytest.mark.parametrize("K", [80, 272, 384])
def test_fp8_scales_stay_in_their_blocks(M, E, N, K):
    """A block's scale that is no number touches that block's columns only, and
    an infinite one makes infinities of its sign, also where the row's last
    columns fill no pair of blocks."""
    q, s, w, ws = _case8(M, E, N, K, M + K)
    q, w = (torch.where(t.float() == 0, 1.0, t.float()).abs().to(FP8) for t in (q, w))
    ends = _ends(_spread_counts(M, E, K))
    want = G.grouped_mm_fp8(q, s, w, ws, ends)
    first, last = next((a, b) for a, b in O.groups(ends.tolist(), M) if b > a)
    e = [b > a for a, b in O.groups(ends.tolist(), M)].index(True)
    for block in range(ws.shape[1]):
        for value in (float("nan"), float("inf")):
            bad = ws.clone()
            bad[e, block, block % ws.shape[2]] = value
            got = G.grouped_mm_fp8(q, s, w, bad, ends)
            at = torch.zeros((M, N), dtype=torch.bool, device=DEV)
            at[first:last, 128 * block:128 * block + 128] = True
            assert torch.equal(got[~at], want[~at])
            assert bool(got[at].isnan().all() if value != value else got[at].isposinf().all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("per", [60, 130])
def test_large_tiles_in_a_graph_and_again(per, fp8):
    """Replayed with other ends, beside eager calls: the same bytes each time."""
    E, N, K = 24, 1800, 400
    M = E * per
    ins = _case8(M, E, N, K, 70) if fp8 else (_randn((M, K), 71), _randn((E, N, K), 72))
    call = G.grouped_mm_fp8 if fp8 else G.grouped_mm
    sets = [_ends(_spread_counts(M - 50 * k, E, k)) for k in range(4)]
    ends = sets[0].clone()
    call(*ins, ends)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(*ins, ends)
    for e in sets + sets[:2]:
        ends.copy_(e)
        want = call(*ins, e)
        out.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(_bits(out), _bits(want))
        assert torch.equal(_bits(call(*ins, e)), _bits(want))


def test_empty():
    w = _randn((2, 16, 32), 50)
    out = G.grouped_mm(torch.empty((0, 32), dtype=BF, device=DEV), w, _ends([0, 0]))
    assert out.shape == (0, 16)
    out = G.grouped_mm(_randn((4, 32), 51), w[:, :0], _ends([2, 2]))
    assert out.shape == (4, 0)


def test_single_rows_of_any_stride():
    """One row, one expert, one output: their strides say nothing."""
    buf = _randn((3, 70000), 80)
    x, ends = buf[1:2, :64], _ends([1])
    w = _randn((1, 1, 64), 81)
    odd = torch.empty(100000, dtype=BF, device=DEV).as_strided((1, 1, 64), (7, 3, 1))
    odd.copy_(w)
    want = G.grouped_mm(x.contiguous(), w, ends)
    assert torch.equal(G.grouped_mm(x, odd, ends), want)
    assert torch.equal(G.grouped_mm(x.as_strided((1, 64), (2 ** 40, 1)), odd, ends), want)
    q, s, w8, ws = _case8(1, 1, 1, 64, 82)
    want = G.grouped_mm_fp8(q, s, w8, ws, ends)
    assert torch.equal(G.grouped_mm_fp8(
        q.as_strided((1, 64), (2 ** 40, 1)), s.as_strided((1, 1), (2 ** 40, 1)),
        w8.as_strided((1, 1, 64), (9, 5, 1)), ws, ends), want)


def test_refusals():
    x, w, ends = _randn((6, 64), 60), _randn((2, 16, 64), 61), _ends([3, 3])
    q, s, w8, ws = _case8(6, 2, 16, 64, 62)
    for bad in (lambda: G.grouped_mm(x[0], w, ends), lambda: G.grouped_mm(x, w[0], ends),
                lambda: G.grouped_mm(x, w, ends[:1]), lambda: G.grouped_mm(x, w, ends.long()),
                lambda: G.grouped_mm(x[:, :32], w, ends), lambda: G.grouped_mm(x, w.cpu(), ends),
                lambda: G.grouped_mm(x, w, ends.cpu()), lambda: G.grouped_mm(x, w[:0], ends[:0]),
                lambda: G.grouped_mm(x, w.transpose(1, 2).contiguous().transpose(1, 2), ends),
                lambda: G.grouped_mm(x, w, ends, out=torch.empty((6, 17), dtype=BF, device=DEV)),
                lambda: G.grouped_mm(x, w, ends, dtype=F32, out=x[:, :16].contiguous()),
                lambda: G.grouped_mm(x, w, ends, out=x.view(-1)[:96].view(6, 16)),
                lambda: G.grouped_mm_fp8(q, s[:5], w8, ws, ends),
                lambda: G.grouped_mm_fp8(q, s, w8, ws[:, :, :0], ends),
                lambda: G.grouped_mm_fp8(q, s.double(), w8, ws, ends),
                lambda: G.grouped_mm_fp8(q, s.cpu(), w8, ws, ends),
                lambda: G.grouped_mm_fp8(q, s, w8, ws, ends, out=torch.empty((6, 16), device=DEV))):
        with pytest.raises(ValueError):
            bad()
    # out in the rows, the ends or the weights of the call
    slab = torch.zeros(4096, dtype=BF, device=DEV)
    for bad in (lambda: G.grouped_mm(x, slab[:2048].view(2, 16, 64), ends,
                                     out=slab[2000:2096].view(6, 16)),
                lambda: G.grouped_mm_fp8(q, s, slab.view(FP8)[:2048].view(2, 16, 64), ws, ends,
                                         out=slab[1000:1096].view(6, 16)),
                lambda: G.grouped_mm_fp8(q, slab.view(F32)[:6].view(6, 1), w8, ws, ends,
                                         out=slab[8:104].view(6, 16)),
                lambda: G.grouped_mm_fp8(q, s, w8, slab.view(F32)[:2].view(2, 1, 1), ends,
                                         out=slab[:96].view(6, 16))):
        with pytest.raises(ValueError, match="overlaps"):
            bad()
    # more rows or columns than a call counts
    one = torch.zeros(16, dtype=BF, device=DEV)
    for bad in (lambda: G.grouped_mm(one.expand(2 ** 31, 16), one.expand(1, 8, 16), ends[:1]),
                lambda: G.grouped_mm(one.expand(4, 16), one.expand(1, 2 ** 32 + 8, 16), ends[:1]),
                lambda: G.grouped_mm(one[:1].expand(4, 2 ** 32 + 8),
                                     one.as_strided((1, 8, 2 ** 32 + 8), (0, 0, 0)), ends[:1])):
        with pytest.raises((NotImplementedError, ValueError)):
            bad()
    for bad in (lambda: G.grouped_mm(x.float(), w, ends), lambda: G.grouped_mm(x, w.float(), ends),
                lambda: G.grouped_mm(x, w, ends, dtype=torch.float16),
                lambda: G.grouped_mm_fp8(x, s, w8, ws, ends),
                lambda: G.grouped_mm_fp8(q[:, :24], s, w8[:, :, :24], ws, ends),
                lambda: G.grouped_mm(x[:, :4], w[:, :, :4], ends)):
        with pytest.raises(NotImplementedError):
            bad()


# Every kernel by name, so that another choice of kernels cannot leave one untested:
# the kernel, FP8, output type, experts, rows an expert, outputs, columns (large tiles:
# whole pairs of chunks, and columns behind a row's end within one and after a whole one).
KERNELS = [
    (_lib.WISP_GROUPED_FEW, False, BF, 3, 10, 72, 136),
    (_lib.WISP_GROUPED_FEW, False, F32, 3, 10, 75, 136),
    (_lib.WISP_GROUPED_FEW, True, BF, 3, 10, 72, 144),
    (_lib.WISP_GROUPED_TILE_64, False, BF, 4, 100, 264, 200),
    (_lib.WISP_GROUPED_TILE_64, False, F32, 4, 100, 260, 256),
    (_lib.WISP_GROUPED_TILE_64, True, BF, 4, 100, 264, 272),
    (_lib.WISP_GROUPED_TILE_64 | _lib.WISP_GROUPED_NARROW, False, BF, 4, 100, 261, 200),
    (_lib.WISP_GROUPED_TILE_64 | _lib.WISP_GROUPED_NARROW, False, F32, 4, 100, 261, 200),
    (_lib.WISP_GROUPED_TILE_64 | _lib.WISP_GROUPED_NARROW, True, BF, 4, 100, 262, 272),
    (_lib.WISP_GROUPED_TILE_128, False, BF, 60, 5, 1672, 200),
    (_lib.WISP_GROUPED_TILE_128, True, BF, 24, 100, 1800, 400),
    (_lib.WISP_GROUPED_TILE_256, False, F32, 110, 5, 1800, 200),
    (_lib.WISP_GROUPED_TILE_256, True, BF, 110, 5, 1800, 208),
    (_lib.WISP_GROUPED_LARGE_128, False, BF, 24, 100, 1800, 200),
    (_lib.WISP_GROUPED_LARGE_128, False, BF, 24, 90, 1800, 256),
    (_lib.WISP_GROUPED_LARGE_128, False, F32, 24, 100, 1796, 272),
    (_lib.WISP_GROUPED_LARGE_192, False, BF, 24, 130, 1800, 200),
    (_lib.WISP_GROUPED_LARGE_192, False, BF, 24, 125, 1800, 512),
    (_lib.WISP_GROUPED_LARGE_192, False, F32, 24, 130, 1796, 144),
    (_lib.WISP_GROUPED_LARGE_256, True, BF, 24, 200, 1800, 144),
    (_lib.WISP_GROUPED_LARGE_256, True, BF, 24, 200, 1800, 272),
    (_lib.WISP_GROUPED_LARGE_256, True, BF, 24, 200, 1800, 384),
    (_lib.WISP_GROUPED_LARGE_256, True, BF, 24, 130, 1800, 512),
]
_kernels = pytest.mark.parametrize("kernel,fp8,dtype,E,per,N,K", KERNELS)


def _runs(kernel, fp8, dtype, E, M, N, K, out=1 << 20):
    """Asserts that a call of these sizes runs ``kernel``."""
    got = _lib.lib().wisp_grouped_mm_kernel(fp8, E, M, N, K, out, G._DTYPES[dtype])
    assert got == kernel, got


def _inputs(fp8, dtype, M, E, N, K, seed):
    """Rows and weights, and the call over them."""
    if fp8:
        return _case8(M, E, N, K, seed), G.grouped_mm_fp8
    return (_randn((M, K), seed), _randn((E, N, K), seed + 1, BF, 0.1)), \
        lambda *a, **kw: G.grouped_mm(*a, dtype=dtype, **kw)


@_kernels
def test_every_kernel_keeps_values_in_their_rows_and_columns(kernel, fp8, dtype, E, per, N, K):
    """What is no number in other groups' rows and scales, behind the last group, in other
    experts' weights and scales, behind a row's last column and behind the last output
    touches nothing else; a given output keeps its rows behind the last group."""
    M, tail = E * per, 7
    _runs(kernel, fp8, dtype, E, M, N, K)
    counts = _spread_counts(M - tail, E, K)
    counts[1], counts[2] = counts[1] + counts[2], 0   # (an expert that no row is for)
    ends = _ends(counts)
    ins, call = _inputs(fp8, dtype, M, E, N, K, per)
    want = call(*ins, ends)
    kind, pad = (torch.uint8, 0x7f) if fp8 else (BF, float("nan"))
    raw = [t.view(kind) if t.element_size() < 4 else t for t in ins]
    x, w = raw[0], raw[2 if fp8 else 1]
    big_x = torch.full((M, K + 96), pad, dtype=kind, device=DEV)
    big_w = torch.full((E, N + 3, K + 160), pad, dtype=kind, device=DEV)
    big_x[:, :K], big_w[:, :N, :K] = x, w
    big_x[M - tail:], big_w[2] = pad, pad
    if fp8:
        g = ins[1].shape[1]
        big_s = torch.full((M, g + 2), float("nan"), device=DEV)
        big_s[:, :g] = ins[1]
        big_s[M - tail:] = float("inf")
        ws = ins[3].clone()
        ws[2] = float("nan")
        args = big_x.view(FP8)[:, :K], big_s[:, :g], big_w.view(FP8)[:, :N, :K], ws, ends
    else:
        args = big_x[:, :K], big_w[:, :N, :K], ends
    assert torch.equal(_bits(call(*args)), _bits(want))
    out = torch.full((M, N), 7.0, dtype=dtype, device=DEV)
    call(*args, out=out)
    assert torch.equal(_bits(out[:M - tail]), _bits(want[:M - tail]))
    assert bool((out[M - tail:] == 7).all()) and not want[M - tail:].any()
    # one row and one weight row of the largest group, one row of the group's last
    e = int(np.argmax(counts))
    first, n = int(sum(counts[:e])), int(counts[e])
    rows = [first + n // 2, first + n - 1]
    bad = torch.zeros((M, N), dtype=torch.bool, device=DEV)
    bad[rows], bad[first:first + n, N - 2] = True, True
    big_x[rows, K - 1], big_w[e, N - 2, K - 1] = pad, pad
    got = call(*args)
    assert torch.equal(_bits(got[~bad]), _bits(want[~bad])) and got[bad].isnan().all()
    if fp8:   # and scales of a row and of a block of weights
        row, block = first + n // 3, (N - 1) // 128
        big_s[row, g - 1] = float("nan")
        ws[e, block, g - 1] = float("nan")
        bad[row], bad[first:first + n, 128 * block:] = True, True
        got = call(*args)
        assert torch.equal(_bits(got[~bad]), _bits(want[~bad])) and got[bad].isnan().all()


@_kernels
def test_every_kernel_in_a_graph(kernel, fp8, dtype, E, per, N, K):
    """Replayed with other ends, rows, weights and scales in the captured buffers, beside
    eager calls: the eager call's bytes each time."""
    M = E * per
    _runs(kernel, fp8, dtype, E, M, N, K)
    sets = [(*_inputs(fp8, dtype, M, E, N, K, 10 * k)[0], _ends(_spread_counts(M - 3 * k, E, k)))
            for k in range(3)]
    ins, call = [t.clone() for t in sets[0]], _inputs(fp8, dtype, 1, 1, 8, 16, 0)[1]
    call(*ins)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(*ins)
    for new in sets + sets[:2]:
        for t, v in zip(ins, new):
            t.copy_(v)
        want = call(*new)
        out.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(_bits(out), _bits(want))


@_kernels
def test_every_kernel_against_rows_of_their_own(kernel, fp8, dtype, E, per, N, K):
    """Rows of a group and the same rows in calls of their own (1, 16, 17 and 60 of them,
    one expert): each within its bound of the exact values, so within two of each other."""
    M = E * per
    _runs(kernel, fp8, dtype, E, M, N, K)
    counts = _spread_counts(M, E, per)
    ins, call = _inputs(fp8, dtype, M, E, N, K, per + 5)
    got = call(*ins, _ends(counts))
    e = int(np.argmax(counts))
    first, n = int(sum(counts[:e])), int(counts[e])
    if fp8:
        x, w = _values8(ins[0][first:first + n], ins[1][first:first + n], ins[2][e:e + 1],
                        ins[3][e:e + 1])
    else:
        x, w = _f64(ins[0][first:first + n]), _f64(ins[1][e:e + 1])
    want, bound = O.grouped_mm(x, w, [n], DOT8 if fp8 else 0.0)
    _near(got[first:first + n], want, bound, dtype)
    bound = 2 * (bound + (O.BF16 if dtype == BF else O.STEP) * (np.abs(want) + bound) + O.TINY)
    for rows in (1, 16, 17, 60):
        for at in {0, n // 2, max(n - rows, 0)}:
            part = slice(first + at, first + min(at + rows, n))
            mine = [t[part] if i < (2 if fp8 else 1) else t[e:e + 1] for i, t in enumerate(ins)]
            alone = call(*mine, _ends([part.stop - part.start]))
            off = np.abs(_f64(alone) - _f64(got[part]))
            assert np.all(off <= bound[at:at + rows])


@_kernels
@pytest.mark.parametrize("at", [1, 2, 4])
def test_outputs_from_any_element_on(kernel, fp8, dtype, E, per, N, K, at):
    """A given output at any element of a larger buffer: its values within their bound, and
    what lies before and behind it as it was."""
    M, few = E * per, 16
    _runs(kernel, fp8, dtype, E, M, N, K)
    counts = _spread_counts(M - 5, E, per)
    ins, call = _inputs(fp8, dtype, M, E, N, K, per + 9)
    slab = torch.full((M * N + 2 * few,), 7.0, dtype=dtype, device=DEV)
    assert slab.data_ptr() % 16 == 0
    out = slab[at:at + M * N].view(M, N)
    want = call(*ins, _ends(counts))
    call(*ins, _ends(counts), out=out)
    # rows that the same kernel stores: the same bytes; those of another: twice the bound
    if dtype == F32 or at % 2 == 0 or kernel == _lib.WISP_GROUPED_FEW:
        assert torch.equal(_bits(out[:M - 5]), _bits(want[:M - 5]))
    else:
        e = int(np.argmax(counts))
        first, n = int(sum(counts[:e])), int(counts[e])
        part = slice(first, first + n)
        x, w = _values8(ins[0][part], ins[1][part], ins[2][e:e + 1], ins[3][e:e + 1]) if fp8 \
            else (_f64(ins[0][part]), _f64(ins[1][e:e + 1]))
        _near(out[part], *O.grouped_mm(x, w, [n], DOT8 if fp8 else 0.0), dtype)
    assert bool((slab[:at] == 7).all()) and bool((out[M - 5:] == 7).all())
    assert bool((slab[at + M * N:] == 7).all())


def test_a_single_expert_s_strides_say_nothing():
    """One expert: weights and block scales any distance from the next."""
    q, s, w, ws = _case8(20, 1, 40, 64, 90)
    ends = _ends([18])
    want = G.grouped_mm_fp8(q, s, w, ws, ends)
    far = [t.as_strided(t.shape, (2 ** 58, *t.stride()[1:])) for t in (w, ws)]
    assert torch.equal(G.grouped_mm_fp8(q, s, far[0], far[1], ends), want)
