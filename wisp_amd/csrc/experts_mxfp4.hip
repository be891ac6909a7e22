// SwiGLU experts over MXFP4 weights (format: mxfp4.h), bf16 activations:
//   act[p] = bf16(silu(W13[s][:I] x[t]) * (W13[s][I:] x[t]))   p = (t, k), s = slots[p]
//   y[p]   = W2[s] act[p]                                        (fp32)
//   out[t] = bf16(sum_{k ascending} w[t,k] * y[p])
// The products run on the bf16 matrix instruction with fp32 sums.  A weight
// becomes its bf16 value, which is exact, in registers on its way into the
// instruction: one conversion instruction gives two values with their scale
// applied.
//
// Small and middle calls (mx_grouped_kernel) are bound by the stream of weights,
// large ones (mx_tile_kernel) by the matrix instructions and what feeds them.
// Measured (us, w13 + w2): Qwen3, 32 tokens 38 + 24 (4.9 and 3.9 TB/s of
// weights; w2's rows are three stages, behind one that only loads), 512 tokens
// 57 + 40; Mixtral, 6 tokens 76 + 50 (5.4 and 4.1); Qwen3, 8192 tokens 452 + 284
// (910 and 730 TFLOP/s; w2 also writes 537 MB of y), Mixtral, 1000 tokens 576 +
// 285 (820 and 820).
#include <math.h>

#include <algorithm>

#include "dma_pipeline.h"
#include "experts_mxfp4.h"
#include "mxfp4.h"
#include "tile_pipeline.h"

namespace wisp {

int experts_mfma_combine(int T, int H, int K, const float* topk_w, const int32_t* slots,
                         int nslots, const void* work, void* out, hipStream_t st);

namespace {

using mx::f32x4;
using mx::u32x4;

constexpr int kChunk = 128;               // k columns of a chunk: four blocks of each row
constexpr int kSub = 2;                   // chunks of a stage
constexpr int kStageK = kSub * kChunk;    // k columns of a stage: 128 bytes of a row's codes
constexpr int kTokBytes = kChunk * 2;     // of a token row, a chunk
constexpr int kTokPerCopy = 1024 / kTokBytes;

// A block of WR waves: each holds NG tiles of 16 weight rows against NT token
// tiles of 16.
template <int WR_, int NG_, int NT_>
struct Shape {
  static constexpr int WR = WR_, NG = NG_, NT = NT_;
  static constexpr int kRows = WR * NG * 16;
  static constexpr int kToks = NT * 16;                   // of a pass
  static constexpr int NC = kToks / kTokPerCopy / WR;     // token copies of a wave and chunk
  static_assert(NC * kTokPerCopy * WR == kToks, "token copies split evenly");
  static constexpr int kPart = kToks * kTokBytes;         // a chunk's tokens
  static constexpr int kWaveW = NG * 16 * 128;            // a wave's codes of a stage
};

// Where the 16-byte pieces of row r stand: piece b at b ^ swizzle(r), in
// 256-byte token rows and in the block tiles' 64-byte code rows.  Lane l reads
// row l % 16 at a piece that depends on l / 16, and one cycle of a 16-byte LDS
// read serves groups of four lanes of different l / 16 together, so pieces
// that differ by l / 16 must not meet between such groups.  The row's own
// number as the swizzle does: 17 to 41 % of the LDS cycles were bank
// conflicts, now none in the grouped kernel and 9 % in the tiles.  Measured
// (us a call): Qwen3, 512 tokens 111.7 -> 108.7, Mixtral, 1000 873 -> 855.
__device__ __attribute__((always_inline)) inline int token_swizzle(int r) {
  return (r & 3) << 2 | (r >> 2 & 3);
}
__device__ __attribute__((always_inline)) inline int code_swizzle(int r) {
  return (r >> 2 & 1) * 3 ^ (r >> 3 & 1);
}

struct GroupedArgs {
  const uint16_t* A;  // token matrix: x (w13) or act (w2)
  int H, I, K, P;
  const int32_t* lists;
  const int32_t* counts;
  const uint8_t* W;
  size_t w_stride;
  const uint8_t* S;
  size_t s_stride;
  void* out;
  int splits;  // of the k range (w2): split z writes its part of y, [P][H], at z * P * H
};

// g / (1 + e^-g), its last few float32 bits apart: act is rounded to bf16.
// (The exponential's argument is clamped where e^-g is 0 or infinite anyway,
// so that an infinite g gives what the formula does; what t's rounding left
// enters as a factor near 1, which leaves an infinite power one.)  Against
// common.h's silu (us a call): Qwen3, 512 tokens 107 / 111, 8192 tokens 798 to
// 804 / 810 to 825, Mixtral, 1000 tokens 824 to 828 / 834 to 839.
__device__ inline float silu_fast(float g) {
  constexpr float kLog2e = 1.44269502f, kLog2eLow = 1.92596299e-8f, kLn2 = 0.693147182f;
  const float n = __builtin_amdgcn_fmed3f(-g, -104.f, 89.f);
  const float t = n * kLog2e;
  const float low = fmaf(n, kLog2e, -t) + n * kLog2eLow;
  const float e = __builtin_amdgcn_exp2f(t) * fmaf(kLn2, low, 1.f);
  return g * __builtin_amdgcn_rcpf(1.f + e);
}

// bf16(silu(g) * u) of four consecutive columns, one 8-byte store at p.  The
// rounding is the matrix instruction's: its operands are bf16.  Against 64 bits
// the output's error is 2.3e-3 of its norm with it and 1.7e-3 without (the
// output's own rounding alone, as in the two launches for a few tokens, whose
// act is float32).
__device__ inline void store_act4(uint16_t* p, const f32x4& g, const f32x4& u) {
  uint32_t h[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) h[q] = bf16_rne(silu_fast(g[q]) * u[q]);
  *reinterpret_cast<uint2*>(p) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// One block's products for the tokens of one slot, a pass of up to kToks of
// them at a time, in stages of 256 k columns.
//
// Weights go through registers one stage ahead: eight lanes read the 128
// bytes of a row (lanes that each read a row of their own, as the matrix
// operand wants them, cost the address unit 64 cycles a load instead of 16
// and hold a stream of weights at 3 TB/s), then into the wave's own part of
// LDS, 16-byte block b of row r at position b ^ (r / 2 % 8), and back in operand
// order: lane l holds row l % 16 of a tile, block l / 16 of a chunk, the
// operands of four matrix instructions, step j over
// k = 32 (l / 16) + 8 j .. + 7.  Lane l loads the scales of the wave's row l.
//
// Token rows are copied to LDS asynchronously one chunk ahead, 256 bytes of
// each, its pieces swizzled (token_swizzle).
//
// kOdd: rows that are not whole stages.  Blocks past a row's end read as
// zeros, and each lane loads its own blocks' scales.
template <typename Sh, bool kW13, bool kOdd>
struct Tile {
  static constexpr int NG = Sh::NG, NT = Sh::NT, NC = Sh::NC;
  static constexpr int per = kW13 ? NG / 2 : NG;  // tiles of output columns of a wave
  static constexpr int NL = 2 * NG;               // code loads of a stage
  static constexpr int NS = kOdd ? kSub * NG : kSub;  // words of scales
  static constexpr int kLoads = NL + (kOdd ? NS : 1);
  static_assert(NG == 4, "a lane for each weight row of the wave");
  const GroupedArgs& a;
  unsigned char* tlds;
  unsigned char* wlds;  // this wave's
  const int32_t* list;
  int wave, lane, q, Kdim, nblk, chunks, N, n0;
  int from, to;       // this block's chunks, whole stages but for a row's end
  mx::Buffer W, S;    // the slot's codes and scales
  uint32_t tile0[NG]; // first weight row of each tile (wave-uniform)
  uint32_t scale0;    // byte of the first scale of the wave's row `lane`

  // Byte of the scale of this lane's block of chunk c in tile g (kOdd).
  __device__ __attribute__((always_inline)) uint32_t scale_at(int g, int c) const {
    return (tile0[g] + (lane & 15)) * (uint32_t)nblk + max(min(c * 4 + q, nblk - 1), 0);
  }

  // A stage's codes, row 8 (n % 2) + l / 8 of tile n / 2, and scale words.
  struct Weights {
    u32x4 w[NL];
    uint32_t s[NS];
  };
  __device__ __attribute__((always_inline)) void load_codes(int n, int c, Weights& b) const {
    const uint32_t rowb = (uint32_t)nblk * mx::kBlockBytes;
    const int blk = c * 4 + (lane & 7);
    // (nothing past the range's end, also in the stage after the last)
    const uint32_t v = blk < min(nblk, to * 4) ? (uint32_t)(lane >> 3) * rowb + blk * mx::kBlockBytes : 1u << 31;
    b.w[n] = mx::load16_nt(W, v, (tile0[n / 2] + n % 2 * 8) * rowb);
  }
  __device__ __attribute__((always_inline)) void load_scales(int c, Weights& b) const {
    if constexpr (kOdd) {
#pragma unroll
      for (int i = 0; i < NS; ++i)
        b.s[i] = mx::load4(S, scale_at(i / kSub, c + i % kSub) & ~3u);
    } else {
      const auto two = mx::load8(S, c < chunks ? scale0 + c * 4 : 1u << 31);
      b.s[0] = two[0], b.s[1] = two[1];
    }
  }

  // Token copies of a pass: their rows, and this lane's piece of each in chunk 0.
  struct Tokens {
    uint32_t row[NC];
    int piece;
  };
  __device__ __attribute__((always_inline)) void copy(int c, const Tokens& t,
                                                      unsigned char* stage) const {
    // (before the first chunk the first, past a row's end its last piece once
    // more: no product uses it)
    const int b = kOdd ? min(max(c, 0) * 16 + t.piece, Kdim / 8 - 1)
                       : max(min(c, chunks - 1), 0) * 16 + t.piece;
    const unsigned char* src = reinterpret_cast<const unsigned char*>(a.A) + b * 16;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      dma::dma16(src + (uint64_t)t.row[i] * (uint32_t)(Kdim * 2),
                 stage + (i * Sh::WR + wave) * 1024);
  }

  // A wave's codes of a chunk in operand order, their scales, and the operands
  // of step 0.
  struct Operands {
    u32x4 codes[NG], v0[NG];
    float scale[NG];
  };
  __device__ __attribute__((always_inline)) void put(const Weights& w) const {
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int r = n * 8 + (lane >> 3);
      *reinterpret_cast<u32x4*>(wlds + r * 128 + (((lane & 7) ^ (r >> 1 & 7)) << 4)) = w.w[n];
    }
  }
  template <int h>
  __device__ __attribute__((always_inline)) void get(int c, const uint32_t (&s)[NS],
                                                     Operands& o) const {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int r = g * 16 + (lane & 15);
      o.codes[g] = *reinterpret_cast<const u32x4*>(
          wlds + r * 128 + (((h * 4 + q) ^ (r >> 1 & 7)) << 4));
      o.scale[g] = __uint_as_float(kOdd ? mx::scale_of(s[g * kSub + h], scale_at(g, c + h) & 3)
                                        : mx::scale_of(__shfl((int)s[h], r), q));
    }
  }

  // Half h of the stage from chunk c on, its tokens in rds; the next chunk's
  // token copies, into wrs, are under way meanwhile, and with h = 0 the next
  // stage's weights, into w.  While the matrix instructions of step j run, the
  // operands of step j + 1 are made, and during the last step the weight
  // operands of the next half.  (wrs and rds are distinct, which the compiler
  // has to know.  It also tells only eight copy instructions of a kernel apart,
  // and waits for all copies before an LDS read if there are more: hence one
  // place for all copies, with a turn of the loop for the first.)
  template <int h>
  __device__ __attribute__((always_inline)) void half(int c, unsigned char* __restrict__ wrs,
                                                      const unsigned char* __restrict__ rds,
                                                      const Tokens& tok, uint32_t (&s)[NS],
                                                      Weights& w, Operands& o,
                                                      f32x4 (&acc)[NG][NT]) const {
    // this chunk's tokens have landed: all loads but the youngest, the weights
    dma::wait_vm<h == 0 ? 0 : kLoads>();
    dma::lds_barrier();
    // (six token tiles leave no registers for a second set of operands: with one,
    // made behind the last tile, 6 to 14 us of 160 to 310 a call less in spills)
    constexpr bool kOne = NT > 5;
    u32x4 t[NT], v1[NG];
    // (what stands past a row's end may be an infinity)
    const bool none = kOdd && (c + h) * 4 + q >= nblk;
    auto token = [&](int i, int j) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(rds + (i * 16 + (lane & 15)) * kTokBytes +
                                                      (((q * 4 + j) ^ token_swizzle(lane)) << 4));
      return none ? u32x4{} : v;
    };
#pragma unroll
    for (int i = 0; i < NT; ++i) t[i] = token(i, 0);
    copy(c + h + 1, tok, wrs);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32x4(&v)[NG] = kOne || j % 2 == 0 ? o.v0 : v1;
      u32x4(&vn)[NG] = kOne || j % 2 == 1 ? o.v0 : v1;
      if (j == 3) {
        if constexpr (h == 1) {
          put(w);
#pragma unroll
          for (int i = 0; i < NS; ++i) s[i] = w.s[i];
          get<0>(c + kSub, s, o);
        } else {
          get<1>(c, s, o);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int g = 0; g < NG; ++g) acc[g][i] = mx::mfma(v[g], t[i], acc[g][i]);
        if (j < 3) t[i] = token(i, j + 1);
        // the operands made behind tile i
        const bool late = kOne || j == 3;
        const int g0 = late ? (i == NT - 1 ? 0 : NG) : i * NG / NT;
        const int g1 = late ? NG : (i + 1) * NG / NT;
#pragma unroll
        for (int g = g0; g < g1; ++g) vn[g] = mx::bf16_of(o.codes[g][(j + 1) & 3], o.scale[g]);
        // (all loads at once would fill the address unit's queue)
        if (h == 0 && j < 2) {
#pragma unroll
          for (int n = (j * NT + i) * NL / (2 * NT); n < (j * NT + i + 1) * NL / (2 * NT); ++n)
            load_codes(n, c + kSub, w);
          if (j == 1 && i == NT - 1) load_scales(c + kSub, w);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  __device__ __attribute__((always_inline)) void pass(int m0, int mrows) const {
    Weights w = {};
    Operands o = {};
    uint32_t s[NS] = {};
    Tokens tok;
    static_assert(Sh::WR * kTokPerCopy % 16 == 0, "a lane's rows have one swizzle");
    tok.piece = (lane & 15) ^ token_swizzle(wave * kTokPerCopy + (lane >> 4));
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int p = list[m0 + min((i * Sh::WR + wave) * kTokPerCopy + (lane >> 4), mrows - 1)];
      tok.row[i] = kW13 ? p / a.K : p;
    }
    f32x4 acc[NG][NT];
    auto clear = [&] {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[g][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    clear();
    // The first turn loads; what it computes is dropped.  (No range is empty:
    // the grid's splits are w2_splits' or one.)
#pragma unroll 1
    for (int c = from - kSub; c < to; c += kSub) {
      if (c == from) clear();
      half<0>(c, tlds + Sh::kPart, tlds, tok, s, w, o, acc);
      half<1>(c, tlds, tlds + Sh::kPart, tok, s, w, o, acc);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = i * 16 + (lane & 15);
      if (r >= mrows) continue;
      const int p = list[m0 + r];
#pragma unroll
      for (int g = 0; g < per; ++g) {
        const int n = n0 + g * 16;
        if (n >= N) break;
        if constexpr (kW13)
          store_act4((uint16_t*)a.out + (size_t)p * N + n + q * 4, acc[g][i], acc[g + per][i]);
        else
          *reinterpret_cast<f32x4*>((float*)a.out + ((size_t)blockIdx.z * a.P + p) * N + n +
                                    q * 4) = acc[g][i];
      }
    }
  }
};

// Grid (panel, slot, split).
template <typename Sh, bool kW13, bool kOdd>
__global__ __launch_bounds__(64 * Sh::WR) __attribute__((amdgpu_waves_per_eu(Sh::NT < 3 ? 3 : 2))) void
mx_grouped_kernel(GroupedArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char tlds[];
  __shared__ __attribute__((aligned(16))) unsigned char wlds[Sh::WR * Sh::kWaveW];
  const int s = blockIdx.y;
  const int M = a.counts[s];
  if (M == 0) return;
  Tile<Sh, kW13, kOdd> t{a, tlds};
  t.list = a.lists + (size_t)s * a.P;
  t.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  t.wlds = wlds + t.wave * Sh::kWaveW;
  t.lane = threadIdx.x & 63;
  t.q = t.lane >> 4;
  t.Kdim = kW13 ? a.H : a.I, t.nblk = t.Kdim / mx::kBlock;
  t.chunks = (t.nblk + 3) / 4;
  const int stages = (t.chunks + kSub - 1) / kSub;
  const int span = (stages + (int)gridDim.z - 1) / (int)gridDim.z * kSub;
  t.from = blockIdx.z * span, t.to = min(t.from + span, t.chunks);
  t.N = kW13 ? a.I : a.H;
  t.n0 = (blockIdx.x * Sh::WR + t.wave) * t.per * 16;
  const uint32_t blocks = (uint32_t)(kW13 ? 2 * a.I : a.H) * (uint32_t)t.nblk;
  t.W = mx::buffer(a.W + (size_t)s * a.w_stride, blocks * mx::kBlockBytes);
  t.S = mx::buffer(a.S + (size_t)s * a.s_stride, blocks);  // a multiple of four
#pragma unroll
  for (int g = 0; g < Sh::NG; ++g)  // (tiles past the end repeat the last)
    t.tile0[g] = (g < t.per ? 0 : a.I) + min(t.n0 + g % t.per * 16, t.N - 16);
  uint32_t row = t.tile0[0];
#pragma unroll
  for (int g = 1; g < Sh::NG; ++g) row = t.q == g ? t.tile0[g] : row;
  t.scale0 = (row + (t.lane & 15)) * (uint32_t)t.nblk;
#pragma unroll 1
  for (int m0 = 0; m0 < M; m0 += Sh::kToks) t.pass(m0, min(M - m0, Sh::kToks));
}

// ---------------------------------------------------------------------------
// Large calls: the same products in tiles of 256 weight rows (w13: 128 gate
// and 128 up rows) by up to 128, 160 or 192 tokens of a slot, eight waves in persistent
// blocks, one per CU: wave (wr, wt) holds 64 rows against the token tiles wt,
// wt + 2, ... of 16.  Stages are single chunks; the last chunk of a tile
// already loads the first of the next.  The matrix instructions and the k
// order of every output are those of the kernel above, so the bytes are too.
// ---------------------------------------------------------------------------
template <int NT_>
struct BigShape {
  static constexpr int WR = 4, WT = 2, NG = 4, NT = NT_;
  static constexpr int kWaves = WR * WT;
  static constexpr int kRows = WR * NG * 16;
  static constexpr int kToks = WT * NT * 16;
  static constexpr int NC = kToks / kTokPerCopy / kWaves;  // token copies of a wave and chunk
  static constexpr int kPart = kToks * kTokBytes;
  static constexpr int kWaveW = NG * 16 * 64;              // a wave's codes of a chunk
  static constexpr int kW = 2 * kPart;
  static constexpr int kTable = kW + kWaves * kWaveW;
  static constexpr int kLds = kTable + (int)sizeof(tile::Table);
};

template <typename Big, bool kW13>
struct BigTile {
  static constexpr int NG = Big::NG, NT = Big::NT, NC = Big::NC;
  static constexpr int per = kW13 ? NG / 2 : NG;
  const GroupedArgs& a;
  unsigned char* lds;
  unsigned char* wlds;
  int wave, lane, wr, wt, q, Kdim, nblk, chunks, N;

  tile::Range tokens;
  struct Source {
    uint32_t src[NC];  // this lane's piece of each token copy's row
    mx::Buffer W, S;
    uint32_t tile0[NG];
    uint32_t scale;  // byte of the first scale of the wave's row `lane`
  };
  struct Weights {
    u32x4 w[NG];
    uint32_t s;
  };

  __device__ __attribute__((always_inline)) int row0(const tile::Work& w) const {
    return (w.panel * Big::WR + wr) * per * 16;
  }
  // The pairs behind this wave's token copies: lane 4 i + n holds that of row
  // n of copy i.
  __device__ __attribute__((always_inline)) int pairs(const tile::Work& w) const {
    static_assert(NC * kTokPerCopy <= 64, "a lane for each row of a wave's copies");
    const int r = ((lane >> 2) * Big::kWaves + wave) * kTokPerCopy + (lane & 3);
    return a.lists[(size_t)w.slot * a.P + w.m0 + min(r, w.mrows - 1)];
  }
  __device__ __attribute__((always_inline)) void source(const tile::Work& w, int pr,
                                                        Source& s) const {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int r = (i * Big::kWaves + wave) * kTokPerCopy + q;
      const int p = __shfl(pr, i * kTokPerCopy + q);
      s.src[i] = (uint32_t)(kW13 ? p / a.K : p) * (uint32_t)(Kdim * 2) +
                 (((lane & 15) ^ token_swizzle(r)) << 4);
    }
    const uint32_t blocks = (uint32_t)(kW13 ? 2 * a.I : a.H) * (uint32_t)nblk;
    s.W = mx::buffer(a.W + (size_t)w.slot * a.w_stride, blocks * mx::kBlockBytes);
    s.S = mx::buffer(a.S + (size_t)w.slot * a.s_stride, blocks);
#pragma unroll
    for (int g = 0; g < NG; ++g)
      s.tile0[g] = (g < per ? 0 : a.I) + min(row0(w) + g % per * 16, N - 16);
    uint32_t row = s.tile0[0];
#pragma unroll
    for (int g = 1; g < NG; ++g) row = q == g ? s.tile0[g] : row;
    s.scale = (row + (lane & 15)) * (uint32_t)nblk;
  }
  // Chunk c's token copy i into a stage.
  __device__ __attribute__((always_inline)) void copy(int i, int c, const Source& s,
                                                      unsigned char* stage) const {
    tile::copy16(tokens, s.src[i], c * kTokBytes, stage + (i * Big::kWaves + wave) * 1024);
  }
  // Chunk c's codes of row tile g, four lanes for the 64 bytes of a row; its
  // scales, lane l those of the wave's row l.
  __device__ __attribute__((always_inline)) void load(int g, int c, const Source& s,
                                                      Weights& b) const {
    const uint32_t rowb = (uint32_t)nblk * mx::kBlockBytes;
    const uint32_t v = (uint32_t)(lane >> 2) * rowb + (c * 4 + (lane & 3)) * mx::kBlockBytes;
    b.w[g] = mx::load16(s.W, v, s.tile0[g] * rowb);
  }
  __device__ __attribute__((always_inline)) void load_scales(int c, const Source& s,
                                                             Weights& b) const {
    b.s = mx::load4(s.S, s.scale + c * 4);
  }

  // A wave's codes of a chunk in operand order, their scales, and the operands
  // of step 0.
  struct Operands {
    u32x4 codes[NG], v0[NG];
    float scale[NG];
  };
  // Through the wave's own LDS (code_swizzle).
  __device__ __attribute__((always_inline)) void put(const Weights& w) const {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int r = g * 16 + (lane >> 2);
      *reinterpret_cast<u32x4*>(wlds + r * 64 + (((lane & 3) ^ code_swizzle(r)) << 4)) = w.w[g];
    }
  }
  __device__ __attribute__((always_inline)) void get(uint32_t s, Operands& o) const {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int r = g * 16 + (lane & 15);
      o.codes[g] = *reinterpret_cast<const u32x4*>(wlds + r * 64 + ((q ^ code_swizzle(r)) << 4));
      o.scale[g] = __uint_as_float(mx::scale_of(__shfl((int)s, r), q));
    }
  }

  // One chunk's products from stage rds and operands o, with the loads of
  // chunk c of `src`.  While the matrix instructions of step j run, the token
  // and weight operands of step j + 1 are made, and during the last step the
  // weight operands of the next chunk, so that only its first token operands
  // are waited for behind the barrier.  The loads go out a few at a time: all
  // together they fill the address unit's queue, and the wave waits there
  // instead of computing (80 of 476 us at the Qwen3
  // 8192-token chunk's w13).
  // For the same reason nothing here is skipped for a tile that is not full:
  // a branch's LDS reads are all waited for where it ends.  (The compiler adds
  // four small loops: it does not see that a code load's row offset, tile0 *
  // rowb, is the wave's.)
  __device__ __attribute__((always_inline)) void step(unsigned char* __restrict__ wrs,
                                                      const unsigned char* __restrict__ rds, int c,
                                                      const Source& src, Weights& w, Operands& o,
                                                      f32x4 (&acc)[NG][NT]) const {
    u32x4 t[NT], v1[NG];
    auto token = [&](int i, int j) {
      return *reinterpret_cast<const u32x4*>(
          rds + ((i * Big::WT + wt) * 16 + (lane & 15)) * kTokBytes +
          (((q * 4 + j) ^ token_swizzle(lane)) << 4));
    };
#pragma unroll
    for (int i = 0; i < NT; ++i) t[i] = token(i, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32x4(&v)[NG] = j & 1 ? v1 : o.v0;
      u32x4(&vn)[NG] = j & 1 ? o.v0 : v1;
      if (j == 3) {
        put(w);
        get(w.s, o);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int g = 0; g < NG; ++g) acc[g][i] = mx::mfma(v[g], t[i], acc[g][i]);
        if (j < 3) t[i] = token(i, j + 1);
        if (j < 3 ? i < NG : i >= NT - NG) {
          const int g = j < 3 ? i : i - (NT - NG);
          vn[g] = mx::bf16_of(o.codes[g][(j + 1) & 3], o.scale[g]);
        }
        // one load behind each tile: the weights, then the token copies
        const int n = j * NT + i;
        static_assert(NG + 1 + NC <= 3 * NT, "the loads go out before step 3 needs them");
        if (n < NG) load(n, c, src, w);
        if (n == NG) load_scales(c, src, w);
        if (n > NG && n <= NG + NC) copy(n - NG - 1, c, src, wrs);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

template <typename Big, bool kW13>
__global__ __launch_bounds__(64 * Big::kWaves)
__attribute__((amdgpu_waves_per_eu(2, 2))) void mx_tile_kernel(GroupedArgs a, int nslots) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  tile::Table* tab = reinterpret_cast<tile::Table*>(lds + Big::kTable);
  BigTile<Big, kW13> t{a, lds};
  t.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  t.lane = threadIdx.x & 63;
  t.wr = t.wave / Big::WT, t.wt = t.wave % Big::WT, t.q = t.lane >> 4;
  t.wlds = lds + Big::kW + t.wave * Big::kWaveW;
  t.Kdim = kW13 ? a.H : a.I, t.nblk = t.Kdim / mx::kBlock, t.chunks = t.nblk / 4;
  t.N = kW13 ? a.I : a.H;
  t.tokens = {a.A, (uint32_t)(kW13 ? a.P / a.K : a.P) * (uint32_t)(t.Kdim * 2)};
  constexpr int cols = kW13 ? Big::kRows / 2 : Big::kRows;
  const int npanels = (t.N + cols - 1) / cols;
  if (t.wave == 0) tile::fill_table(tab, a.counts, nslots, Big::kToks);
  __syncthreads();
  int j = 0;
  auto take = [&](tile::Work& w) {
    const bool found = tile::find_work(tab, tile::work_of(blockIdx.x, j++), nslots, npanels, &w);
    w.slot = __builtin_amdgcn_readfirstlane(w.slot);
    w.panel = __builtin_amdgcn_readfirstlane(w.panel);
    w.m0 = __builtin_amdgcn_readfirstlane(w.m0);
    w.mrows = __builtin_amdgcn_readfirstlane(w.mrows);
    return (bool)__builtin_amdgcn_readfirstlane(found);
  };
  tile::Work cur, next;
  if (!take(cur)) return;
  typename BigTile<Big, kW13>::Source src;
  typename BigTile<Big, kW13>::Weights w = {};
  int stage = 0;
  bool have = true;  // `next` is a work
  next = cur;
  f32x4 acc[Big::NG][Big::NT];
  int np = t.pairs(next);
  typename BigTile<Big, kW13>::Operands o = {};
  // Turn c computes chunk c of `cur` and loads chunk c + 1, or the first of
  // `next` (of `cur` once more if there is none).  What the first turn
  // computes, from zero operands, is dropped.
  for (int c = t.chunks - 1, first = 1;;) {
    const bool last = c + 1 == t.chunks;
    if (last && have) t.source(next, np, src);
    dma::wait_vm<0>();
    dma::lds_barrier();
    t.step(lds + (stage ^ 1) * Big::kPart, lds + stage * Big::kPart, last ? 0 : c + 1, src, w, o,
           acc);
    stage ^= 1;
    if (!last) {
      ++c;
      continue;
    }
    if (!first) {
      const int32_t* list = a.lists + (size_t)cur.slot * a.P + cur.m0;
      const int n0 = t.row0(cur);
#pragma unroll
      for (int i = 0; i < Big::NT; ++i) {
        const int r = (i * Big::WT + t.wt) * 16 + (t.lane & 15);
        if (r >= cur.mrows) continue;
        const int p = list[r];
#pragma unroll
        for (int g = 0; g < t.per; ++g) {
          const int n = n0 + g * 16;
          if (n >= t.N) break;
          if constexpr (kW13)
            store_act4((uint16_t*)a.out + (size_t)p * t.N + n + t.q * 4, acc[g][i],
                       acc[g + t.per][i]);
          else
            *reinterpret_cast<f32x4*>((float*)a.out + (size_t)p * t.N + n + t.q * 4) = acc[g][i];
        }
      }
    }
    if (!have) break;
    cur = next;
    have = take(next);
    if (have) np = t.pairs(next);
    c = 0;
    first = 0;
#pragma unroll
    for (int g = 0; g < Big::NG; ++g)
#pragma unroll
      for (int i = 0; i < Big::NT; ++i) acc[g][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

template <typename Sh, bool kW13, bool kOdd>
hipError_t launch_grouped(const GroupedArgs& a, dim3 grid, hipStream_t st, hipEvent_t e0,
                          hipEvent_t e1) {
  constexpr unsigned lds = 2 * Sh::kPart;
  static_assert(lds + Sh::WR * Sh::kWaveW <= 160 * 1024, "LDS per block");
  static std::atomic<uint64_t> big{0};
  const hipError_t e =
      allow_lds(&mx_grouped_kernel<Sh, kW13, kOdd>, lds + Sh::WR * Sh::kWaveW, lds, &big);
  if (e != hipSuccess) return e;
  launch_timed_lds(mx_grouped_kernel<Sh, kW13, kOdd>, grid, dim3(64 * Sh::WR), lds, st, e0, e1, a);
  return hipSuccess;
}

// Calls of at least this many pairs a slot take the block tiles: from here the
// blocks above pass over most slots' weights twice.  Measured, the blocks above
// against tiles (us a call): Qwen3 177 / 212 at 72 pairs a slot, 211 / 213 at
// 80; Mixtral 325 / 449 at 80, 508 / 457 at 100.  84 is where Qwen3's times meet;
// Mixtral's meet at about 95, and below it takes longer than in the blocks: 317 /
// 411 to 446 at 84, 361 / 444 at 87, 397 / 461 at 90, 438 / 445 at 93.  (Pairs
// without a slot count: the slots are in device memory.)
constexpr int kTilePairs = 84;

// The pairs of a call's slots: their mean, the deviation that a random router
// gives them, and how many deviations the fullest of so many slots has more.
struct Spread {
  double mean, dev, fullest;
  Spread(int P, int slots, int K)
      : mean((double)P / slots),
        dev(sqrt(mean * (1 - std::min(1.0, (double)K / slots)))),
        fullest(0.93 + 0.22 * log2((double)slots)) {}
};

// How long a call's tiles of this shape take, in token tiles of a wave (a
// chunk costs a wave about two token tiles besides its products): halfway
// between their rounds of 256 blocks and their share of a round, since not every
// block of the last round has a tile.  Measured, 128 / 160 / 192 tokens (us a
// call): Qwen3 217 / 225 / 246 at 96 pairs a slot, 256 / 232 / 253 at 112, 355 /
// 295 / 268 at 144, 372 / 407 / 387 at 187, 488 / 441 / 482 at 256, 884 / 857 /
// 785 at 512; Mixtral 545 / 488 / 517 at 128, 690 / 751 / 582 at 175, 728 / 806
// / 893 at 212, 1038 / 812 / 901 at 250.
template <typename Big>
double tile_cost(const Spread& s, int slots, int panels) {
  auto of = [](double m) { return ceil(std::max(m, 1.0) / Big::kToks); };
  const double tiles = (of(s.mean - s.dev) + of(s.mean) + of(s.mean + s.dev) +
                        0.5 * of(s.mean + s.fullest * s.dev)) / 3.5 * slots;
  const double rounds = tiles * panels / tile::kBlocks;
  return 0.5 * (ceil(rounds) + std::max(rounds, 1.0)) * (Big::NT + 2);
}

template <typename Big, bool kW13>
hipError_t launch_tiles(const GroupedArgs& a, int nslots, hipStream_t st, hipEvent_t e0,
                        hipEvent_t e1) {
  static_assert(Big::kLds <= 160 * 1024, "LDS per block");
  static std::atomic<uint64_t> big{0};
  const hipError_t e = allow_lds(&mx_tile_kernel<Big, kW13>, Big::kLds, Big::kLds, &big);
  if (e != hipSuccess) return e;
  launch_timed_lds(mx_tile_kernel<Big, kW13>, dim3(tile::kBlocks), dim3(64 * Big::kWaves),
                   Big::kLds, st, e0, e1, a, nslots);
  return hipSuccess;
}

// The token tiles (of 16) of a pass of the grouped kernel: those by which the
// slots' passes take the least.  A pass with more tiles takes longer (kPass, the
// times of calls of one pass over many experts), one with fewer leaves more
// slots a second pass over their weights.  Where the blocks do not fill the GPU
// the fullest slot alone counts.  Measured, NT / NT + 1 (us a call; M: Mixtral,
// else Qwen3): 8 pairs a slot 81 / 81, 9: 89 / 81; 20: 97 / 98, 22: 105 / 99;
// 34: 113 / 115, 40: 144 / 117; 44: 121 / 129, 56: 169 / 139, M 50: 224 / 244,
// M 54: 273 / 247; 64: 163 / 169, 72: 207 / 177, M 64: 262 / 302, M 72:
// 331 / 302.  The fullest slot: 24 experts of 1056 x 352 at 87 pairs a slot,
// 4 / 6 tiles 73 / 98.
int token_tiles(const Spread& s, int64_t blocks) {
  constexpr double kPass[] = {1, 1.08, 1.25, 1.45, 1.7, 2};
  int best = 1;
  double least = 0;
  for (int nt = 1; nt <= 6; ++nt) {
    double passes = 0;
    for (double z : {-1.3, -0.5, 0.5, 1.3})
      passes += ceil(std::max(1.0, s.mean + (blocks < 512 ? s.fullest : z) * s.dev) / (16 * nt));
    passes += ceil((s.mean + s.fullest * s.dev) / (16 * nt));
    const double cost = passes * kPass[nt - 1];
    if (nt == 1 || cost < least) best = nt, least = cost;
  }
  return best;
}

template <bool kW13>
hipError_t launch_product(const GroupedArgs& a, int nslots, hipStream_t st, hipEvent_t e0,
                          hipEvent_t e1) {
  const int spread = std::min(a.P, nslots);
  const Spread pairs(a.P, spread, a.K);
  auto go = [&](auto shape) {
    using Sh = decltype(shape);
    constexpr int per = Sh::kRows / (kW13 ? 2 : 1);
    const dim3 grid(((kW13 ? a.I : a.H) + per - 1) / per, nslots, a.splits);
    return (kW13 ? a.H : a.I) % kStageK ? launch_grouped<Sh, kW13, true>(a, grid, st, e0, e1)
                                        : launch_grouped<Sh, kW13, false>(a, grid, st, e0, e1);
  };
  // (the tiles' token offsets are 32 bits wide)
  const uint64_t bytes = (uint64_t)(kW13 ? a.P / a.K : a.P) * (kW13 ? a.H : a.I) * 2;
  const int panels = kW13 ? (a.I + 127) / 128 : (a.H + 255) / 256;
  if (a.splits == 1 && a.P >= kTilePairs * spread && (kW13 ? a.H : a.I) % kChunk == 0 &&
      nslots <= kMaxExperts && bytes < 1ull << 32) {
    const double c4 = tile_cost<BigShape<4>>(pairs, spread, panels),
                 c5 = tile_cost<BigShape<5>>(pairs, spread, panels),
                 c6 = tile_cost<BigShape<6>>(pairs, spread, panels);
    return c4 < std::min(c5, c6) ? launch_tiles<BigShape<4>, kW13>(a, nslots, st, e0, e1)
           : c5 < c6             ? launch_tiles<BigShape<5>, kW13>(a, nslots, st, e0, e1)
                                 : launch_tiles<BigShape<6>, kW13>(a, nslots, st, e0, e1);
  }
  switch (token_tiles(pairs, (int64_t)panels * spread * a.splits)) {
    case 1: return go(Shape<4, 4, 1>{});
    case 2: return go(Shape<4, 4, 2>{});
    case 3: return go(Shape<4, 4, 3>{});
    case 4: return go(Shape<4, 4, 4>{});
    case 5: return go(Shape<4, 4, 5>{});
    default: return go(Shape<4, 4, 6>{});
  }
}

// out[t, h] = bf16(sum_k w[t,k] * sum_z y[z, (t,k), h]), k and z ascending;
// pairs without a slot are passed over.  Grid (ceil(H / 1024), T).
__global__ __launch_bounds__(256) void mx_combine_kernel(const float* __restrict__ y, int splits,
                                                         int P, int H, int K, int nslots,
                                                         const float* __restrict__ topk_w,
                                                         const int32_t* __restrict__ slots,
                                                         uint16_t* __restrict__ out) {
  const int t = blockIdx.y, h = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (h >= H) return;
  f32x4 acc{0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < K; ++k) {
    const int p = t * K + k, s = slots[p];
    if (s < 0 || s >= nslots) continue;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    for (int z = 0; z < splits; ++z)
      v += *reinterpret_cast<const f32x4*>(y + ((size_t)z * P + p) * H + h);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(topk_w[p], v[e], acc[e]);
  }
  *reinterpret_cast<uint2*>(out + (size_t)t * H + h) =
      make_uint2(bf16_rne(acc[0]) | (uint32_t)bf16_rne(acc[1]) << 16,
                 bf16_rne(acc[2]) | (uint32_t)bf16_rne(acc[3]) << 16);
}

// Splits of w2's k range: a call whose panels are too few to fill the GPU (16
// of 256 rows at H 4096), and whose block tiles would be, splits it into parts
// of at least four stages but for the last, which is not empty (25 stages in six
// parts of five would leave one).  It goes by the whole call alone, for the
// bytes depend on it.  Measured, 1 / 4 splits, Mixtral: w2 at 6 tokens 100 / 49
// us; a call, where unsplit is block tiles, at 336 tokens 540 / 446, 400 544 /
// 446, 512 559 / 503, 640 604 / 560, 700 615 / 584 to 615, 768 727 / 752.
int w2_splits(int T, int K, int H, int I, int nslots) {
  const int panels = (H + 255) / 256;
  const double mean = (double)T * K / nslots;
  if (mean >= kTilePairs && ceil(mean / BigShape<6>::kToks) * nslots * panels >= tile::kBlocks)
    return 1;
  const double blocks = mx::distinct(T, K, nslots) * panels;
  const int splits = std::max(1, std::min((int)ceil(512 / blocks), I / (4 * kStageK)));
  const int stages = (I + kStageK - 1) / kStageK, span = (stages + splits - 1) / splits;
  return (stages + span - 1) / span;
}

// Work buffer (pair lists, counts, y).
struct Work {
  size_t lists, counts, y, total;
  Work(int P, int H, int nslots, int splits) {
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    lists = 0;
    counts = up((size_t)nslots * P * 4);
    y = counts + up((size_t)nslots * 4);
    total = y + up((size_t)splits * P * H * 4);
  }
};

}  // namespace

// How a call is computed, by what it is as a whole: its tokens, shape and number
// of experts, never by the groups or slots it is paged in, so that paged and
// resident runs of one batch give the same bytes.
Mxfp4Plan mxfp4_plan(int T, int K, int H, int I, int experts) {
  if (mxfp4_few(T, K, H, I, experts)) return {true, 1};
  return {false, w2_splits(std::max(T, 1), K, H, I, experts)};
}

// Work buffer of (part of) a call of T tokens over nslots slots.
size_t mxfp4_work_bytes(const Mxfp4Plan& plan, int T, int K, int H, int I, int nslots) {
  if (T < 1 || K < 1 || H < 1 || I < 1 || nslots < 1) return 0;
  return plan.few ? mxfp4_few_bytes(T * K, I) : Work(T * K, H, nslots, plan.splits).total;
}

// Why the MXFP4 kernels do not cover a call, or null.
const char* mxfp4_unsupported(int H, int I, int K) {
  if (H < mx::kBlock || I < mx::kBlock || H % mx::kBlock || I % mx::kBlock)
    return "hidden and intermediate sizes must be multiples of 32";
  if ((uint64_t)H * I >= 1ull << 31) return "an expert's matrices exceed 2^31 values";
  if (K < 1 || K > kMaxTopK) return "top_k outside [1, 64]";
  return nullptr;
}

namespace {

int check_work(const Mxfp4Plan& plan, int T, int K, int H, int I, int nslots, const void* work,
               size_t work_bytes) {
  if (nslots <= 65535 && work && work_bytes >= mxfp4_work_bytes(plan, T, K, H, I, nslots) &&
      (uintptr_t)work % 256 == 0)
    return WISP_OK;
  wisp_set_last_error("work buffer missing, misaligned or too small", "MXFP4 experts");
  return WISP_ERR_INVALID;
}

}  // namespace

int experts_mxfp4(const Mxfp4Plan& plan, const void* x, int T, int H, int I, int K,
                  const float* topk_w, const int32_t* slots, int nslots, const void* w13,
                  size_t w13_stride, const void* s13, size_t s13_stride, const void* w2,
                  size_t w2_stride, const void* s2, size_t s2_stride, void* act, void* out,
                  void* work, size_t work_bytes, hipStream_t st, const StageEvents* ev) {
  if (T == 0) return WISP_OK;
  const int rc = check_work(plan, T, K, H, I, nslots, work, work_bytes);
  if (rc != WISP_OK) return rc;
  if (plan.few)
    return mxfp4_few_layer(x, nullptr, 0, 0, nullptr, T, H, I, K, const_cast<float*>(topk_w),
                           const_cast<int32_t*>(slots), nslots, w13, w13_stride, s13, s13_stride,
                           w2, w2_stride, s2, s2_stride, work, out, st, ev);
  const int P = T * K;
  const int splits = plan.splits;
  const Work wk(P, H, nslots, splits);
  int32_t* lists = (int32_t*)((char*)work + wk.lists);
  int32_t* counts = (int32_t*)((char*)work + wk.counts);
  launch_gather(slots, P, nslots, lists, counts, st);
  const GroupedArgs a13{(const uint16_t*)x, H, I, K, P, lists, counts, (const uint8_t*)w13,
                        w13_stride, (const uint8_t*)s13, s13_stride, act, 1};
  const GroupedArgs a2{(const uint16_t*)act, H, I, K, P, lists, counts, (const uint8_t*)w2,
                       w2_stride, (const uint8_t*)s2, s2_stride, (char*)work + wk.y, splits};
  WISP_HIP_TRY((launch_product<true>(a13, nslots, st, ev ? ev->ev[0] : nullptr,
                                     ev ? ev->ev[1] : nullptr)));
  WISP_HIP_TRY((launch_product<false>(a2, nslots, st, ev ? ev->ev[2] : nullptr,
                                      ev ? ev->ev[3] : nullptr)));
  WISP_HIP_TRY(hipGetLastError());
  if (splits == 1) return experts_mfma_combine(T, H, K, topk_w, slots, nslots, work, out, st);
  hipLaunchKernelGGL(mx_combine_kernel, dim3((H + 1023) / 1024, T), dim3(256), 0, st,
                     (const float*)((char*)work + wk.y), splits, P, H, K, nslots, topk_w, slots,
                     (uint16_t*)out);
  WISP_HIP_TRY(hipGetLastError());
  return WISP_OK;
}

// Routing (logits [T][experts]) and the experts, expert e in slot e.  `forward`:
// the layer-call counter or null.
int layer_mxfp4(const Mxfp4Plan& plan, const void* x, const void* logits, int logits_dtype,
                int renorm, int64_t* forward, int T, int H, int I, int K, float* topk_w,
                int32_t* ids, int experts, const void* w13, size_t w13_stride, const void* s13,
                size_t s13_stride, const void* w2, size_t w2_stride, const void* s2,
                size_t s2_stride, void* act, void* out, void* work, size_t work_bytes,
                hipStream_t st, const StageEvents* ev) {
  if (T > 0 && plan.few) {
    const int rc = check_work(plan, T, K, H, I, experts, work, work_bytes);
    if (rc != WISP_OK) return rc;
    return mxfp4_few_layer(x, logits, logits_dtype, renorm, forward, T, H, I, K, topk_w, ids,
                           experts, w13, w13_stride, s13, s13_stride, w2, w2_stride, s2, s2_stride,
                           work, out, st, ev);
  }
  const int rc = wisp_route_topk_softmax(logits, logits_dtype, T, experts, K, renorm, topk_w, ids,
                                         forward, (wisp_stream_t)st);
  if (rc != WISP_OK) return rc;
  return experts_mxfp4(plan, x, T, H, I, K, topk_w, ids, experts, w13, w13_stride, s13, s13_stride,
                       w2, w2_stride, s2, s2_stride, act, out, work, work_bytes, st, ev);
}

}  // namespace wisp

namespace {

// Checks of the two entry points below.
int check_call(const void* x, int T, int H, int I, int K, int nslots, const void* w13,
               size_t w13_stride, const void* s13, size_t s13_stride, const void* w2,
               size_t w2_stride, const void* s2, size_t s2_stride, const void* act,
               const void* out, const char* where) {
  using namespace wisp;
  if (T < 0 || nslots < 1 || (T > 0 && (!x || !w13 || !w2 || !s13 || !s2 || !act || !out)) ||
      (int64_t)T * (K > 0 ? K : 1) > 0x7fffffff) {
    wisp_set_last_error("missing buffer or bad count", where);
    return WISP_ERR_INVALID;
  }
  const char* why = mxfp4_unsupported(H, I, K);
  if (!why && ((uintptr_t)w13 % 16 || (uintptr_t)w2 % 16 || w13_stride % 16 || w2_stride % 16 ||
               (uintptr_t)x % 16 || (uintptr_t)act % 16 || (uintptr_t)out % 16 ||
               (uintptr_t)s13 % 4 || (uintptr_t)s2 % 4 || s13_stride % 4 || s2_stride % 4))
    why = "weights, their strides and the activations must be 16-byte aligned, scales and their "
          "strides 4-byte";
  if (why) {
    wisp_set_last_error(why, where);
    return WISP_ERR_UNSUPPORTED;
  }
  const size_t n = (size_t)H * I;
  if (nslots > 1 && (w13_stride < n || w2_stride < n / 2 || s13_stride < n / 16 ||
                     s2_stride < n / 32)) {
    wisp_set_last_error("experts overlap: a stride is below an expert's bytes", where);
    return WISP_ERR_INVALID;
  }
  return WISP_OK;
}

}  // namespace

extern "C" size_t wisp_moe_mxfp4_work_bytes(int T, int K, int H, int I, int nslots) {
  if (T < 1 || K < 1 || H < 1 || I < 1 || nslots < 1 || (int64_t)T * K > 0x7fffffff) return 0;
  return wisp::mxfp4_work_bytes(wisp::mxfp4_plan(T, K, H, I, nslots), T, K, H, I, nslots);
}

extern "C" int wisp_moe_experts_mxfp4(const void* x, int T, int H, int I, int K,
                                      const float* topk_w, const int32_t* slots, int nslots,
                                      const void* w13, size_t w13_stride, const void* s13,
                                      size_t s13_stride, const void* w2, size_t w2_stride,
                                      const void* s2, size_t s2_stride, void* act, void* out,
                                      void* work, size_t work_bytes, wisp_stream_t stream) {
  using namespace wisp;
  const char* where = "wisp_moe_experts_mxfp4";
  const int rc = check_call(x, T, H, I, K, nslots, w13, w13_stride, s13, s13_stride, w2, w2_stride,
                            s2, s2_stride, act, out, where);
  if (rc != WISP_OK) return rc;
  if (T > 0 && (!topk_w || !slots)) {
    wisp_set_last_error("missing routing", where);
    return WISP_ERR_INVALID;
  }
  return experts_mxfp4(mxfp4_plan(T, K, H, I, nslots), x, T, H, I, K, topk_w, slots, nslots, w13,
                       w13_stride, s13, s13_stride, w2, w2_stride, s2, s2_stride, act, out, work,
                       work_bytes, (hipStream_t)stream, nullptr);
}

extern "C" int wisp_moe_layer_mxfp4(const void* x, const void* logits, int logits_dtype, int T,
                                    int H, int I, int E, int K, int renormalize, float* topk_w,
                                    int32_t* topk_ids, const void* w13, size_t w13_stride,
                                    const void* s13, size_t s13_stride, const void* w2,
                                    size_t w2_stride, const void* s2, size_t s2_stride, void* act,
                                    void* out, void* work, size_t work_bytes,
                                    wisp_stream_t stream) {
  using namespace wisp;
  const char* where = "wisp_moe_layer_mxfp4";
  int rc = check_call(x, T, H, I, K, E, w13, w13_stride, s13, s13_stride, w2, w2_stride, s2,
                      s2_stride, act, out, where);
  if (rc != WISP_OK) return rc;
  if (E > kMaxExperts || K > E || (T > 0 && (!logits || !topk_w || !topk_ids)) ||
      (logits_dtype != WISP_F32 && logits_dtype != WISP_BF16)) {
    wisp_set_last_error("invalid routing arguments", where);
    return WISP_ERR_INVALID;
  }
  const Mxfp4Plan plan = mxfp4_plan(T, K, H, I, E);
  return layer_mxfp4(plan, x, logits, logits_dtype, renormalize, nullptr, T, H, I, K, topk_w,
                     topk_ids, E, w13, w13_stride, s13, s13_stride, w2, w2_stride, s2, s2_stride,
                     act, out, work, work_bytes, (hipStream_t)stream, nullptr);
}
