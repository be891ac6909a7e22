// The whole MoE layer over MXFP4 experts (format: mxfp4.h) for a few tokens,
// in two launches: [route + w13 per pair] [w2 + combine].
//   act[p] = silu(W13[s][:I] x[t]) * (W13[s][I:] x[t])   p = (t, k), s = its expert
//   out[t] = bf16(sum_{k ascending} w[t,k] * (W2[s] act[p]))
// Such a call is bound by its launches and by the chain of dependent loads in
// each, so every pair has blocks of its own (an expert of two tokens is read
// twice, the second time from cache), the sums are vector dot products (no
// trip through LDS into a matrix operand's order), and act stays in float32
// between the launches.  Measured (us, w13 + w2; a whole call in a graph):
// Qwen3, one token 7.5 + 6.2; 12.5 (20 MB of weights, 4 us at the rate of a large
// copy), 512 x 256 with 16 experts 3.9 + 4.0; 7.3.
#include <algorithm>
#include <type_traits>

#include "experts_mxfp4.h"
#include "mxfp4.h"
#include "route_core.h"

namespace wisp {
namespace {

using mx::u32x4;

// Sum over each 8-lane half row, the same bits in every lane of it.
__device__ inline float row8_sum_f32(float v) {
  v += dpp_f32<0xB1>(v);   // quad_perm [1,0,3,2]
  v += dpp_f32<0x4E>(v);   // quad_perm [2,3,0,1]
  v += dpp_f32<0x141>(v);  // row_half_mirror
  return v;
}

// act of a pair: 16-byte piece j (0..7) of column block b at piece
// j * (I / 32) + b, so that lanes with consecutive blocks read contiguously.
__device__ inline size_t act_at(int i, int nblk) {
  return ((size_t)(i % mx::kBlock / 4) * nblk + i / mx::kBlock) * 4 + i % 4;
}

// ---------------------------------------------------------------------------
// w13: block (16 columns, pair), a wave for 4 columns, 16 lanes for the gate
// row and the up row of one.  A lane takes one column block in 16, four at a
// time (2048 columns a turn), its x in registers: the first turn's is loaded
// before the routing, which needs nothing of it.
// ---------------------------------------------------------------------------
constexpr int kTurn = 4;

template <typename TL>
struct FewRoute {
  const TL* logits;  // [T][E]
  int E, renorm;
  float* w;          // [T][K]
  int32_t* ids;
  int64_t* forward;  // layer-call counter or null
};
struct FewSlots {
  const int32_t* slots;  // [T][K]
  int nslots;
};

struct FewW13 {
  const uint16_t* x;
  int H, I, K;
  const uint8_t* W;
  size_t w_stride;
  const uint8_t* S;
  size_t s_stride;
  float* act;
};

template <typename Src, int VALS>
__global__ __launch_bounds__(256) void mx_few_w13_kernel(FewW13 a, Src src) {
  __shared__ RoutePos pos;
  __shared__ int32_t chosen;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int pair = blockIdx.y, t = pair / a.K, k = pair - t * a.K;
  const int l16 = lane & 15, nblk = a.H / mx::kBlock;
  const u32x4* xr = reinterpret_cast<const u32x4*>(a.x + (size_t)t * a.H);
  u32x4 x[kTurn][4];
  auto load_x = [&](int b0) {
#pragma unroll
    for (int c = 0; c < kTurn; ++c) {
      const int b = min(b0 + c * 16 + l16, nblk - 1);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[c][j] = xr[b * 4 + j];
    }
  };
  int s;
  if constexpr (std::is_same_v<Src, FewSlots>) {
    s = scalar_word(src.slots + pair);
    load_x(0);
    if (s < 0 || s >= src.nslots) return;  // (w2 does not read this pair's act)
  } else {
    float raw[VALS];
    if (wave == 0) route_load_logits(src.logits + (size_t)t * src.E, src.E, lane, raw);
    load_x(0);
    if (wave == 0) {
      const bool writes = blockIdx.x == 0 && k == a.K - 1;
      float w;
      int id;
      route_token_loaded<VALS>(raw, src.E, k + 1, src.renorm, lane, true, &w, &id, pos, nullptr,
                               writes);
      if (lane == k) chosen = id;
      if (writes && lane < a.K) {
        src.w[(size_t)t * a.K + lane] = w;
        src.ids[(size_t)t * a.K + lane] = id;
      }
      if (writes && t == 0 && lane == 0 && src.forward) src.forward[0] += 1;
    }
    block_lds_sync();
    s = __builtin_amdgcn_readfirstlane(chosen);
  }
  const int i = (blockIdx.x * 4 + wave) * 4 + (lane >> 4);  // I is a multiple of 32
  const uint32_t blocks = 2u * a.I * nblk;  // a multiple of four
  const mx::Buffer W = mx::buffer(a.W + (size_t)s * a.w_stride, blocks * mx::kBlockBytes);
  const mx::Buffer S = mx::buffer(a.S + (size_t)s * a.s_stride, blocks);
  const uint32_t row[2] = {(uint32_t)i * nblk, (uint32_t)(a.I + i) * nblk};
  float sum[2] = {0.f, 0.f};
  for (int b0 = 0; b0 < nblk; b0 += 16 * kTurn) {
    u32x4 w[2][kTurn];
    uint32_t sc[2][kTurn];
#pragma unroll
    for (int c = 0; c < kTurn; ++c) {
      const int b = b0 + c * 16 + l16;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        w[r][c] = mx::load16_nt(W, b < nblk ? (row[r] + b) * mx::kBlockBytes : 1u << 31, 0);
        sc[r][c] = mx::load4(S, (row[r] + min(b, nblk - 1)) & ~3u);
      }
    }
    if (b0 > 0) load_x(b0);
#pragma unroll
    for (int c = 0; c < kTurn; ++c) {
      const int b = b0 + c * 16 + l16;
      if (b < nblk) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float scale = __uint_as_float(mx::scale_of(sc[r][c], (row[r] + b) & 3));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const mx::Pairs v = mx::pairs_of(w[r][c][j], scale);
#pragma unroll
            for (int n = 0; n < 4; ++n) sum[r] = mx::dot2(v.p[n], x[c][j][n], sum[r]);
          }
        }
      }
    }
  }
  const float g = row16_sum_f32(sum[0]), u = row16_sum_f32(sum[1]);
  if (l16 == 0) a.act[(size_t)pair * a.I + act_at(i, a.I / mx::kBlock)] = silu(g) * u;
}

// ---------------------------------------------------------------------------
// w2 + combine: block of 8 output columns, 8 lanes for the row of each.  Its
// eight waves take the pairs in turn; where a token has fewer than eight, the
// k range of a pair is split over kSplit = 8 / K of them (by K alone, so that
// the bytes of a token do not depend on the call's other tokens).  act
// passes through the wave's own LDS: 1024 columns at a time.
// ---------------------------------------------------------------------------
constexpr int kW2Waves = 8;
constexpr int kW2Turn = 4;                    // column blocks of a lane at a time
constexpr int kWindow = 8 * kW2Turn;          // column blocks of a wave at a time
constexpr int kFewPairs = 128;

struct FewW2 {
  const float* act;
  int H, I, K, P, nslots, splits;
  const float* topk_w;
  const int32_t* slots;
  const uint8_t* W;
  size_t w_stride;
  const uint8_t* S;
  size_t s_stride;
  uint16_t* out;
};

__global__ __launch_bounds__(64 * kW2Waves) void mx_few_w2_kernel(FewW2 a) {
  __shared__ __attribute__((aligned(16))) float win[kW2Waves][8 * kWindow * 4];
  __shared__ float part[kFewPairs * 8];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int l8 = lane & 7, h0 = blockIdx.x * 8, h = h0 + (lane >> 3);
  const int nblk = a.I / mx::kBlock;
  const int span = (nblk + a.splits - 1) / a.splits;
  const uint32_t blocks = (uint32_t)a.H * nblk, row = (uint32_t)h * nblk;
  float* mine = win[wave];
  for (int job = wave; job < a.P * a.splits; job += kW2Waves) {
    const int p = job / a.splits, from = (job - p * a.splits) * span, to = min(from + span, nblk);
    const int s = scalar_word(a.slots + p);
    float sum = 0.f;
    if (s >= 0 && s < a.nslots) {
      const mx::Buffer W = mx::buffer(a.W + (size_t)s * a.w_stride, blocks * mx::kBlockBytes);
      const mx::Buffer S = mx::buffer(a.S + (size_t)s * a.s_stride, blocks);
      const u32x4* ap = reinterpret_cast<const u32x4*>(a.act + (size_t)p * a.I);
      for (int b0 = from; b0 < to; b0 += kWindow) {
        u32x4 w[kW2Turn], v[kW2Turn];
        uint32_t sc[kW2Turn];
#pragma unroll
        for (int c = 0; c < kW2Turn; ++c) {
          const int b = b0 + c * 8 + l8;
          w[c] = mx::load16_nt(W, b < to ? (row + b) * mx::kBlockBytes : 1u << 31, 0);
          sc[c] = mx::load4(S, (row + min(b, nblk - 1)) & ~3u);
        }
        // the window's act: eight pieces of kWindow blocks, lane by lane
#pragma unroll
        for (int c = 0; c < kW2Turn; ++c) {
          const int n = c * 64 + lane, j = n / kWindow, b = min(b0 + n % kWindow, nblk - 1);
          v[c] = ap[j * nblk + b];
        }
        wave_lds_sync();  // the window before has been read
#pragma unroll
        for (int c = 0; c < kW2Turn; ++c)
          reinterpret_cast<u32x4*>(mine)[c * 64 + lane] = v[c];
        wave_lds_sync();
#pragma unroll
        for (int c = 0; c < kW2Turn; ++c) {
          if (b0 + c * 8 >= to) break;
          if (b0 + c * 8 + l8 < to) {
            const float scale =
                __uint_as_float(mx::scale_of(sc[c], (row + b0 + c * 8 + l8) & 3));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float f[8];
              mx::f32_of(w[c][j], scale, f);
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const mx::f32x4 y = *reinterpret_cast<const mx::f32x4*>(
                    mine + ((j * 2 + n) * kWindow + c * 8 + l8) * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum = fmaf(f[n * 4 + e], y[e], sum);
              }
            }
          }
        }
      }
    }
    sum = row8_sum_f32(sum);
    if (l8 == 0) part[job * 8 + (lane >> 3)] = sum;
  }
  __syncthreads();
  const int T = a.P / a.K;
  for (int n = threadIdx.x; n < T * 8; n += 64 * kW2Waves) {
    const int t = n >> 3, r = n & 7;
    float acc = 0.f;
    for (int k = 0; k < a.K; ++k) {
      const int p = t * a.K + k, s = a.slots[p];
      if (s < 0 || s >= a.nslots) continue;
      float y = 0.f;
      for (int q = 0; q < a.splits; ++q) y += part[(p * a.splits + q) * 8 + r];
      acc = fmaf(a.topk_w[p], y, acc);
    }
    a.out[(size_t)t * a.H + h0 + r] = bf16_rne(acc);
  }
}

template <typename Src, int VALS>
void launch_w13(const FewW13& a, int P, const Src& src, hipStream_t st, hipEvent_t e0,
                hipEvent_t e1) {
  launch_timed(mx_few_w13_kernel<Src, VALS>, dim3(a.I / 16, P), dim3(256), st, e0, e1, a, src);
}

template <typename TL>
void launch_route_w13(const FewW13& a, int P, const FewRoute<TL>& r, hipStream_t st, hipEvent_t e0,
                      hipEvent_t e1) {
  with_route_vals(r.E, [&](auto vals) {
    launch_w13<FewRoute<TL>, decltype(vals)::value>(a, P, r, st, e0, e1);
  });
}

}  // namespace

// Whether the two launches above serve a call: they read every pair's expert,
// where the grouped GEMM reads every expert once, at a lower rate (small calls:
// 4.3 against 5.0 TB/s of weights) and behind 12 us more of launches.
// Measured, these against the grouped GEMM (us a call): Qwen3 30 / 53 at 5
// tokens, 42 / 58 at 8, 59 / 60 at 12, 67 / 61 at 14; Mixtral 109 / 122 at 3,
// 142 / 132 at 4.
constexpr int kFewTokens = 12;
bool mxfp4_few(int T, int K, int H, int I, int nslots) {
  const int splits = std::max(1, kW2Waves / K);
  if (T > kFewTokens || T * K * splits > kFewPairs) return false;
  const double expert = 3.0 * H * I * 17 / 32;  // bytes
  return T * K * expert / 5.0e6 <= mx::distinct(T, K, nslots) * expert / 4.3e6 + 12;
}

// Bytes of act between the two launches.
size_t mxfp4_few_bytes(int P, int I) { return (size_t)P * I * sizeof(float); }

int mxfp4_few_layer(const void* x, const void* logits, int logits_dtype, int renorm,
                    int64_t* forward, int T, int H, int I, int K, float* topk_w, int32_t* slots,
                    int nslots, const void* w13, size_t w13_stride, const void* s13,
                    size_t s13_stride, const void* w2, size_t w2_stride, const void* s2,
                    size_t s2_stride, void* act, void* out, hipStream_t st, const StageEvents* ev) {
  hipEvent_t e[4] = {};
  for (int i = 0; ev && i < 4; ++i) e[i] = ev->ev[i];
  const int P = T * K;
  const FewW13 a{(const uint16_t*)x, H, I, K, (const uint8_t*)w13, w13_stride,
                 (const uint8_t*)s13, s13_stride, (float*)act};
  if (!logits)
    launch_w13<FewSlots, 2>(a, P, FewSlots{slots, nslots}, st, e[0], e[1]);
  else if (logits_dtype == WISP_F32)
    launch_route_w13(a, P,
                     FewRoute<float>{(const float*)logits, nslots, renorm, topk_w, slots, forward},
                     st, e[0], e[1]);
  else
    launch_route_w13(
        a, P, FewRoute<uint16_t>{(const uint16_t*)logits, nslots, renorm, topk_w, slots, forward},
        st, e[0], e[1]);
  const FewW2 b{(const float*)act, H, I, K, P, nslots, std::max(1, kW2Waves / K), topk_w, slots,
                (const uint8_t*)w2, w2_stride, (const uint8_t*)s2, s2_stride, (uint16_t*)out};
  launch_timed(mx_few_w2_kernel, dim3(H / 8), dim3(64 * kW2Waves), st, e[2], e[3], b);
  WISP_HIP_TRY(hipGetLastError());
  return WISP_OK;
}

}  // namespace wisp
