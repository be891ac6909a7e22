// SwiGLU experts over MXFP4 weights (format: mxfp4.h), bf16 activations:
//   act[p] = bf16(silu(W13[s][:I] x[t]) * (W13[s][I:] x[t]))   p = (t, k), s = slots[p]
//   y[p]   = W2[s] act[p]                                        (fp32)
//   out[t] = bf16(sum_{k ascending} w[t,k] * y[p])
// The products run on the bf16 matrix instruction with fp32 sums.  A weight
// becomes its bf16 value, which is exact, in registers on its way into the
// instruction: one conversion instruction gives two values with their scale
// applied.
#include <algorithm>
#include <type_traits>

#include "dma_pipeline.h"
#include "mxfp4.h"

namespace wisp {

int experts_mfma_combine(int T, int H, int K, const float* topk_w, const int32_t* slots,
                         int nslots, const void* work, void* out, hipStream_t st);
size_t mfma_work_bytes(int T, int K, int H, int nslots);

namespace {

using mx::bf16x8;
using mx::f32x4;
using mx::u32x4;

constexpr int kChunk = 128;               // k columns of a step: four blocks of each row
constexpr int kTokBytes = kChunk * 2;     // of a token row
constexpr int kTokPerCopy = 1024 / kTokBytes;

// A block of WR x WT waves: wave (wr, wt) holds NG tiles of 16 weight rows
// and the NT token tiles of 16 from wt * NT on.
template <int WR_, int WT_, int NG_, int NT_>
struct Shape {
  static constexpr int WR = WR_, WT = WT_, NG = NG_, NT = NT_;
  static constexpr int kWaves = WR * WT;
  static constexpr int kRows = WR * NG * 16;
  static constexpr int kToks = WT * NT * 16;
  static constexpr int kCopies = kToks / kTokPerCopy / kWaves;  // per wave and chunk
  static_assert(kCopies * kTokPerCopy * kWaves == kToks, "token copies split evenly");
  static constexpr int kStage = kToks * kTokBytes;
};

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
};

// The weights of one chunk: a lane's block of each of its row tiles.
template <int NG>
struct Weights {
  u32x4 w[NG];
  uint32_t s[NG];
};

// bf16(silu(g) * u) of four consecutive columns, one 8-byte store at p.
__device__ inline void store_act4(uint16_t* p, const f32x4& g, const f32x4& u) {
  uint32_t h[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) h[q] = bf16_rne(silu(g[q]) * u[q]);
  *reinterpret_cast<uint2*>(p) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// Grid (panel, slot).  Lane l of a wave feeds row l % 16 of a tile, block
// l / 16 of the chunk: its 16 bytes of codes are the operands of four matrix
// instructions, step j over k = 32 (l / 16) + 8 j .. + 7.  Token rows are
// staged in LDS, 256 bytes of each a chunk, 16-byte piece b of row r at
// position b ^ (r % 16).
template <typename Sh, bool kW13, bool kTail>
__global__ __launch_bounds__(64 * Sh::kWaves) void mx_grouped_kernel(GroupedArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  constexpr int NG = Sh::NG, NT = Sh::NT;
  const int s = blockIdx.y;
  const int M = a.counts[s];
  if (M == 0) return;
  const int32_t* list = a.lists + (size_t)s * a.P;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wr = wave / Sh::WT, wt = wave % Sh::WT, q = lane >> 4;
  const int Kdim = kW13 ? a.H : a.I, nblk = Kdim / mx::kBlock;
  const int chunks = (nblk + 3) / 4;
  // first output column of row tile g, and how many columns there are
  const int N = kW13 ? a.I : a.H;
  constexpr int per = kW13 ? NG / 2 : NG;  // tiles of output columns
  const int n0 = (blockIdx.x * Sh::WR + wr) * per * 16;
  const uint8_t* W = a.W + (size_t)s * a.w_stride;
  const uint8_t* S = a.S + (size_t)s * a.s_stride;
  uint32_t row[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int n = min(n0 + g % per * 16, N - 16);  // tiles past the end repeat the last
    row[g] = (uint32_t)((g < per ? 0 : a.I) + n + (lane & 15)) * (uint32_t)nblk;
  }
  auto load = [&](int c, Weights<NG>& b) {
    const int blk = kTail ? min(c * 4 + q, nblk - 1) : c * 4 + q;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      b.w[g] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4*>(W + (size_t)(row[g] + blk) * mx::kBlockBytes));
      b.s[g] = S[row[g] + blk];
    }
  };
  for (int m0 = 0; m0 < M; m0 += Sh::kToks) {
    const int mrows = min(M - m0, Sh::kToks);
    const unsigned char* src[Sh::kCopies];
    int piece[Sh::kCopies];
#pragma unroll
    for (int i = 0; i < Sh::kCopies; ++i) {
      const int r = (i * Sh::kWaves + wave) * kTokPerCopy + (lane >> 4);
      const int p = list[m0 + min(r, mrows - 1)];
      src[i] = reinterpret_cast<const unsigned char*>(a.A + (size_t)(kW13 ? p / a.K : p) * Kdim);
      piece[i] = (lane & 15) ^ (r & 15);
    }
    auto copy = [&](int c, unsigned char* stage) {
#pragma unroll
      for (int i = 0; i < Sh::kCopies; ++i) {
        const int b = kTail ? min(c * 16 + piece[i], Kdim / 8 - 1) : c * 16 + piece[i];
        dma::dma16(src[i] + (size_t)b * 16, stage + (i * Sh::kWaves + wave) * 1024);
      }
    };
    f32x4 acc[NG][NT];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[g][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    Weights<NG> w;
    for (int c = 0; c < chunks; ++c) {
      copy(c, lds);
      load(c, w);
      dma::wait_vm<0>();
      dma::lds_barrier();
      const bool none = kTail && c * 4 + q >= nblk;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8 t[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int r = (wt * NT + i) * 16 + (lane & 15);
          t[i] = *reinterpret_cast<const bf16x8*>(lds + r * kTokBytes +
                                                  (((q * 4 + j) ^ (lane & 15)) << 4));
          if (none) t[i] = bf16x8{};
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const bf16x8 v =
              mx::bf16_of(none ? 0u : w.w[g][j], __uint_as_float((none ? 0u : w.s[g]) << 23));
#pragma unroll
          for (int i = 0; i < NT; ++i)
            acc[g][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, t[i], acc[g][i], 0, 0, 0);
        }
      }
      dma::lds_barrier();
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = (wt * NT + i) * 16 + (lane & 15);
      if (r >= mrows) continue;
      const int p = list[m0 + r];
#pragma unroll
      for (int g = 0; g < per; ++g) {
        const int n = n0 + g * 16;
        if (n >= N) break;
        if constexpr (kW13)
          store_act4((uint16_t*)a.out + (size_t)p * N + n + q * 4, acc[g][i], acc[g + per][i]);
        else
          *reinterpret_cast<f32x4*>((float*)a.out + (size_t)p * N + n + q * 4) = acc[g][i];
      }
    }
  }
}

using Mid = Shape<4, 1, 4, 4>;

template <bool kW13>
void launch_grouped(const GroupedArgs& a, int nslots, hipStream_t st, hipEvent_t e0,
                    hipEvent_t e1) {
  const int cols = kW13 ? a.I : a.H, per = kW13 ? Mid::kRows / 2 : Mid::kRows;
  const dim3 grid((cols + per - 1) / per, nslots);
  if ((kW13 ? a.H : a.I) % kChunk)
    launch_timed_lds(mx_grouped_kernel<Mid, kW13, true>, grid, dim3(64 * Mid::kWaves), Mid::kStage,
                     st, e0, e1, a);
  else
    launch_timed_lds(mx_grouped_kernel<Mid, kW13, false>, grid, dim3(64 * Mid::kWaves),
                     Mid::kStage, st, e0, e1, a);
}

// Work buffer: the layout of the bf16 grouped GEMM's (pair lists, counts, y).
struct Work {
  size_t lists, counts, y;
  Work(int P, int nslots) {
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    lists = 0;
    counts = up((size_t)nslots * P * 4);
    y = counts + up((size_t)nslots * 4);
  }
};

}  // namespace

size_t mxfp4_work_bytes(int T, int K, int H, int nslots) {
  return mfma_work_bytes(T, K, H, nslots);
}

// Why the MXFP4 kernels do not cover a call, or null.
const char* mxfp4_unsupported(int H, int I, int K) {
  if (H < mx::kBlock || I < mx::kBlock || H % mx::kBlock || I % mx::kBlock)
    return "hidden and intermediate sizes must be multiples of 32";
  if ((uint64_t)H * I >= 1ull << 31) return "an expert's matrices exceed 2^31 values";
  if (K < 1 || K > kMaxTopK) return "top_k outside [1, 64]";
  return nullptr;
}

int experts_mxfp4(const void* x, int T, int H, int I, int K, const float* topk_w,
                  const int32_t* slots, int nslots, const void* w13, size_t w13_stride,
                  const void* s13, size_t s13_stride, const void* w2, size_t w2_stride,
                  const void* s2, size_t s2_stride, void* act, void* out, void* work,
                  size_t work_bytes, hipStream_t st, const StageEvents* ev) {
  if (T == 0) return WISP_OK;
  if (nslots > 65535 || !work || work_bytes < mxfp4_work_bytes(T, K, H, nslots) ||
      ((uintptr_t)work) % 256) {
    wisp_set_last_error("work buffer missing, misaligned or too small", "MXFP4 experts");
    return WISP_ERR_INVALID;
  }
  const int P = T * K;
  const Work wk(P, nslots);
  int32_t* lists = (int32_t*)((char*)work + wk.lists);
  int32_t* counts = (int32_t*)((char*)work + wk.counts);
  launch_gather(slots, P, nslots, lists, counts, st);
  const GroupedArgs a13{(const uint16_t*)x, H, I, K, P, lists, counts, (const uint8_t*)w13,
                        w13_stride, (const uint8_t*)s13, s13_stride, act};
  const GroupedArgs a2{(const uint16_t*)act, H, I, K, P, lists, counts, (const uint8_t*)w2,
                       w2_stride, (const uint8_t*)s2, s2_stride, (char*)work + wk.y};
  launch_grouped<true>(a13, nslots, st, ev ? ev->ev[0] : nullptr, ev ? ev->ev[1] : nullptr);
  launch_grouped<false>(a2, nslots, st, ev ? ev->ev[2] : nullptr, ev ? ev->ev[3] : nullptr);
  WISP_HIP_TRY(hipGetLastError());
  return experts_mfma_combine(T, H, K, topk_w, slots, nslots, work, out, st);
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
               (uintptr_t)x % 16 || (uintptr_t)act % 16 || (uintptr_t)out % 16))
    why = "weights, their strides and the activations must be 16-byte aligned";
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

extern "C" size_t wisp_moe_mxfp4_work_bytes(int T, int K, int H, int nslots) {
  return wisp::mxfp4_work_bytes(T, K, H, nslots);
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
  return experts_mxfp4(x, T, H, I, K, topk_w, slots, nslots, w13, w13_stride, s13, s13_stride, w2,
                       w2_stride, s2, s2_stride, act, out, work, work_bytes, (hipStream_t)stream,
                       nullptr);
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
  rc = wisp_route_topk_softmax(logits, logits_dtype, T, E, K, renormalize, topk_w, topk_ids,
                               nullptr, stream);
  if (rc != WISP_OK) return rc;
  return experts_mxfp4(x, T, H, I, K, topk_w, topk_ids, E, w13, w13_stride, s13, s13_stride, w2,
                       w2_stride, s2, s2_stride, act, out, work, work_bytes, (hipStream_t)stream,
                       nullptr);
}
