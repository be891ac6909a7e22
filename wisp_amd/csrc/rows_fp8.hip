// Rows before and between the experts' products: the RMS norm with the
// residual's addition, and the SwiGLU, with outputs in the rows' type or in 8
// bits with scales.
//
//   r = round(x + residual)                      (r = x without a residual)
//   y = r * (mean(r^2) + eps)^(-1/2) * weight    in float32
//   y = silu(h[:I]) * h[I:]                      in float32
//   per group of 128 columns (a row's last one may be shorter):
//     s = max(max|y|, 1e-10) / 448,  q = e4m3fn(y / s), nearest, ties to even
// The codes come from the float32 y: one rounding a value, where a norm that
// writes bfloat16 and a quantiser that reads it make two.  y / s is
// y * (448 / max|y|), one division a group; against a division a value (both
// round twice) only what lies within 2^-22 of a border between two codes differs.
// A group that holds an infinity or a NaN gets NaN codes.
//
// A thread holds eight consecutive values of a row, so a group is 16 lanes
// (its maximum four DPP steps) and every access of a wave one contiguous run.
#include <type_traits>

#include "common.h"

namespace wisp {
namespace {

constexpr int kPer = 8;      // consecutive values a thread holds
constexpr int kGroup = 128;  // columns of a scale
constexpr float kE4m3Max = 448.f;
constexpr float kLeast = 1e-10f;

// Eight consecutive values as they lie in memory.
struct Raw16 {
  uint4 u;
};
struct Raw32 {
  float4 a, b;
};
template <typename T>
struct RawOf;
template <>
struct RawOf<uint16_t> {
  using type = Raw16;
};
template <>
struct RawOf<float> {
  using type = Raw32;
};

// VEC: p is 16-byte aligned and n >= 8.  Otherwise the first n values, zeros
// behind.
template <bool VEC>
__device__ inline Raw16 raw8(const uint16_t* p, int n) {
  if constexpr (VEC) return Raw16{*reinterpret_cast<const uint4*>(p)};
  uint32_t w[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) w[j] = j < n ? p[j] : 0;
  return Raw16{make_uint4(w[0] | (w[1] << 16), w[2] | (w[3] << 16), w[4] | (w[5] << 16),
                          w[6] | (w[7] << 16))};
}
template <bool VEC>
__device__ inline Raw32 raw8(const float* p, int n) {
  if constexpr (VEC)
    return Raw32{reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
  float w[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) w[j] = j < n ? p[j] : 0.f;
  return Raw32{make_float4(w[0], w[1], w[2], w[3]), make_float4(w[4], w[5], w[6], w[7])};
}
__device__ inline void unpack(const Raw16& r, float (&v)[kPer]) {
  const uint32_t w[4] = {r.u.x, r.u.y, r.u.z, r.u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}
__device__ inline void unpack(const Raw32& r, float (&v)[kPer]) {
  v[0] = r.a.x, v[1] = r.a.y, v[2] = r.a.z, v[3] = r.a.w;
  v[4] = r.b.x, v[5] = r.b.y, v[6] = r.b.z, v[7] = r.b.w;
}

template <bool VEC>
__device__ inline void store8(uint16_t* p, int n, const float (&v)[kPer]) {
  if constexpr (VEC) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = (uint32_t)bf16_rne(v[2 * j]) | ((uint32_t)bf16_rne(v[2 * j + 1]) << 16);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < n) p[j] = bf16_rne(v[j]);
  }
}
template <bool VEC>
__device__ inline void store8(float* p, int n, const float (&v)[kPer]) {
  if constexpr (VEC) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < n) p[j] = v[j];
  }
}

// What a value of type T keeps of a float32.
__device__ inline float round_to(float f, const uint16_t*) { return bf16f(bf16_rne(f)); }
__device__ inline float round_to(float f, const float*) { return f; }

// Codes of one group, eight values a lane of 16, all of which come here
// together; a lane behind the row's end holds zeros and has live false.  The
// group's first lane writes the scale.
template <bool VEC>
__device__ inline void quantize8(const float (&y)[kPer], int n, bool live, uint8_t* q,
                                 float* scale) {
  // magnitudes compare as their bits: a NaN is above the infinity
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, false));
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, false));
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xF, 0xF, false));
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xF, 0xF, false));
  const float top = __uint_as_float(max(m, __float_as_uint(kLeast)));
  const float inv = kE4m3Max / top;
  float c[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) c[j] = __builtin_amdgcn_fmed3f(y[j] * inv, -kE4m3Max, kE4m3Max);
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], hi, true);
  if (m >= 0x7f800000u) lo = hi = 0x7f7f7f7f;
  if (!live) return;
  if constexpr (VEC) {
    // (non-temporal: 8192 rows of 4096 in 44.5 us, 47.7 without)
    __builtin_nontemporal_store((uint64_t)(uint32_t)lo | (uint64_t)(uint32_t)hi << 32,
                                reinterpret_cast<uint64_t*>(q));
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < n) q[j] = (uint8_t)((uint32_t)(j < 4 ? lo : hi) >> (8 * (j & 3)));
  }
  if (threadIdx.x % 16 == 0) *scale = top / kE4m3Max;
}

// ---------------------------------------------------------------------------
// The norm
// ---------------------------------------------------------------------------

struct NormArgs {
  const void *x, *residual, *weight;
  void *residual_out, *out;
  uint8_t* q;
  float* scales;
  int64_t rows, x_stride, residual_stride, residual_out_stride;
  int cols, groups;
  float eps;
};

// TPR threads hold a row, PER runs of kPer values each, so that a row is read
// once.  R: the residual's type, void without one; W: the weight's.  A row's
// outputs may be its inputs' memory: a thread writes only what it has read.
template <typename X, typename R, typename W, bool VEC, int TPR, int PER>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void add_rms_norm_kernel(const NormArgs a) {
  constexpr bool kRes = !std::is_void<R>::value;
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / TPR) + threadIdx.x / TPR;
  if (TPR < 256 && row >= a.rows) return;  // (all of a row's threads, so all of a DPP row)
  const X* x = (const X*)a.x + row * a.x_stride;
  typename RawOf<X>::type xr[PER];
  typename RawOf<W>::type wr[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = (i * TPR + t) * kPer;
    if (c < a.cols) xr[i] = raw8<VEC>(x + c, a.cols - c);
  }
  float v[PER][kPer];
  if constexpr (kRes) {
    typename RawOf<R>::type rr[PER];
    const R* res = (const R*)a.residual + row * a.residual_stride;
    R* to = (R*)a.residual_out + row * a.residual_out_stride;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * TPR + t) * kPer;
      if (c < a.cols) rr[i] = raw8<VEC>(res + c, a.cols - c);
    }
    // (in flight with the row: the sum's chain would add their latency)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * TPR + t) * kPer;
      if (c < a.cols) wr[i] = raw8<VEC>((const W*)a.weight + c, a.cols - c);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * TPR + t) * kPer;
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[i][j] = 0.f;
      if (c >= a.cols) continue;
      float r[kPer];
      unpack(xr[i], v[i]);
      unpack(rr[i], r);
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[i][j] = round_to(v[i][j] + r[j], to);
      store8<VEC>(to + c, a.cols - c, v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * TPR + t) * kPer;
      if (c < a.cols) wr[i] = raw8<VEC>((const W*)a.weight + c, a.cols - c);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[i][j] = 0.f;
      if ((i * TPR + t) * kPer < a.cols) unpack(xr[i], v[i]);
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum = __builtin_fmaf(v[i][j], v[i][j], sum);
  if constexpr (TPR == 16) {
    sum = row16_sum_f32(sum);
  } else {
    sum = wave_sum_f32(sum);
    if constexpr (TPR > 64) {
      __shared__ float part[TPR / 64];
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
      block_lds_sync();
      sum = part[0];
#pragma unroll
      for (int i = 1; i < TPR / 64; ++i) sum += part[i];
    }
  }
  const float scale = 1.f / sqrtf(sum / (float)a.cols + a.eps);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = (i * TPR + t) * kPer, n = a.cols - c;
    if (c - (t % 16) * kPer >= a.cols) continue;  // (none of the group's 16 lanes has a value)
    float y[kPer] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n > 0) {
      float w[kPer];
      unpack(wr[i], w);
#pragma unroll
      for (int j = 0; j < kPer; ++j) y[j] = VEC || j < n ? v[i][j] * scale * w[j] : 0.f;
      if (a.out) store8<VEC>((X*)a.out + row * a.cols + c, n, y);
    }
    if (a.q)
      quantize8<VEC>(y, n, n > 0, a.q + row * a.cols + c,
                     a.scales + row * a.groups + c / kGroup);
  }
}

template <typename X, typename R, typename W, bool VEC, int TPR, int PER>
int launch_norm(const NormArgs& a, hipStream_t st) {
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  const int64_t blocks = (a.rows + kThreads / TPR - 1) / (kThreads / TPR);
  if (blocks * kThreads >= (int64_t)1 << 32) {  // (a launch has fewer threads than that)
    wisp_set_last_error("too many rows", "wisp_add_rms_norm");
    return WISP_ERR_UNSUPPORTED;
  }
  hipLaunchKernelGGL((add_rms_norm_kernel<X, R, W, VEC, TPR, PER>), dim3((unsigned)blocks),
                     dim3(kThreads), 0, st, a);
  WISP_HIP_TRY(hipGetLastError());
  return WISP_OK;
}

template <typename X, typename R, typename W>
int norm_of(const NormArgs& a, bool vec, hipStream_t st) {
  // As many threads as hold the row in one or two runs each (more waves wait at a
  // barrier, fewer have too few loads in flight).  us, bf16 with a residual and
  // codes: 65536 rows of 1024 in waves of their own 82.7, in blocks of 256 99.9;
  // 8192 of 4096 44.5 by 256 threads, 52.2 by 64; 2048 of 8192 24.2 by 512, 26.4 by
  // 256; 4096 of 14336 75.2 by 512, 99.4 by 1024 of four runs.  Bound by memory
  // (4.9 to 5.7 TB/s; a 2 GiB copy moves 4.92); few rows by the launch (32 of 2048
  // 3.9 us).
  const int c = a.cols;
  if (vec) {
    if (c <= 128) return launch_norm<X, R, W, true, 16, 1>(a, st);
    if (c <= 512) return launch_norm<X, R, W, true, 64, 1>(a, st);
    if (c <= 1024) return launch_norm<X, R, W, true, 64, 2>(a, st);
    if (c <= 2048) return launch_norm<X, R, W, true, 256, 1>(a, st);
    if (c <= 4096) return launch_norm<X, R, W, true, 256, 2>(a, st);
    if (c <= 8192) return launch_norm<X, R, W, true, 512, 2>(a, st);
    if (c <= 16384) return launch_norm<X, R, W, true, 512, 4>(a, st);
    return launch_norm<X, R, W, true, 1024, 4>(a, st);
  }
  // rows that are not whole, aligned runs: value by value
  if (c <= 512) return launch_norm<X, R, W, false, 64, 1>(a, st);
  if (c <= 2048) return launch_norm<X, R, W, false, 256, 1>(a, st);
  if (c <= 8192) return launch_norm<X, R, W, false, 512, 2>(a, st);
  return launch_norm<X, R, W, false, 1024, 4>(a, st);
}

constexpr int kMaxCols = 1024 * 4 * kPer;

// ---------------------------------------------------------------------------
// The SwiGLU
// ---------------------------------------------------------------------------

// g / (1 + exp(-g)), within some steps of float32 at every g: the hardware's
// exponential of the rounded exponent, times what the rounding left, and the
// hardware's reciprocal with one step of Newton.  The library's functions would
// take twice the instructions, and the vector units would bound the kernel.
// (The exponent is made from g within [-128, 128]: g * log2(e) of the largest g is
// infinite, and what its rounding left is no number.)
// FAR, for gates below kFarGate: 1 + exp(-g) and its reciprocal would leave float32
// before their product with g does, so both are taken 2^64 times smaller and larger; of
// 1 + exp(-g) the 1 is below 2^-123.  From -128 down the value is below 2^-177 |g|: zero,
// and an infinity's no number.  Other gates give the same bytes either way.
constexpr float kFarGate = -86.f;
template <bool FAR>
__device__ inline float silu_fast(float g) {
  // (p is the rounded product everywhere, also in p - 64: what is left is that one's)
#pragma clang fp contract(off)
  constexpr float kLog2e = 1.44269504088896340736f, kRest = 1.92596299e-8f, kLn2 = 0.69314718f;
  const float t = FAR ? __builtin_amdgcn_fmed3f(g, -128.f, 128.f) : fminf(g, 128.f);
  const float p = t * -kLog2e;
  const float rest = __builtin_fmaf(t, -kRest, __builtin_fmaf(t, -kLog2e, -p)) * kLn2;
  const bool far = FAR && g < kFarGate;
  const float e = __builtin_amdgcn_exp2f(far ? p - 64.f : p);
  const float d = 1.f + __builtin_fmaf(e, rest, e);
  float r = __builtin_amdgcn_rcpf(d);
  r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.f), r, r);
  return g * r * (far ? (g <= -128.f ? 0.f : 0x1p-64f) : 1.f);
}

// One group a DPP row of 16 lanes.  65536 rows of 768 in 48 to 50 us (5.0 to 5.3 TB/s), 43 without
// the SiLU's arithmetic: memory and the vector units, which overlap in part.  Two
// or four groups a thread, their loads first: 50 and 52; persistent blocks 51.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void silu_mul_fp8_kernel(const T* __restrict__ h,
                                                           int64_t h_stride, int64_t jobs,
                                                           int inter, int groups,
                                                           uint8_t* __restrict__ q,
                                                           float* __restrict__ scales) {
  const int64_t job = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (job >= jobs) return;  // (all 16 lanes of it)
  const int64_t row = job / groups;
  const int c = (int)(job - row * groups) * kGroup + (threadIdx.x & 15) * kPer;
  const int n = inter - c;
  float y[kPer] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (n > 0) {
    const T* p = h + row * h_stride + c;
    const auto gr = raw8<VEC>(p, n);
    const auto ur = raw8<VEC>(p + inter, n);
    float g[kPer], u[kPer];
    unpack(gr, g);
    unpack(ur, u);
    float least = g[0];
#pragma unroll
    for (int j = 1; j < kPer; ++j) least = fminf(least, g[j]);
    // (a wave without such gates makes no choice for each value: 65536 rows of 768 in
    // 48.1 us, 50.2 with the choices everywhere)
    if (__any(least < kFarGate)) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) y[j] = silu_fast<true>(g[j]) * u[j];
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) y[j] = silu_fast<false>(g[j]) * u[j];
    }
  }
  quantize8<VEC>(y, n, n > 0, q + row * inter + c, scales + job);
}

template <typename T>
void launch_silu(const void* h, int64_t h_stride, int64_t jobs, int inter, int groups, uint8_t* q,
                 float* scales, bool vec, hipStream_t st) {
  const dim3 grid((unsigned)((jobs + 15) / 16));
  if (vec)
    hipLaunchKernelGGL((silu_mul_fp8_kernel<T, true>), grid, dim3(256), 0, st, (const T*)h,
                       h_stride, jobs, inter, groups, q, scales);
  else
    hipLaunchKernelGGL((silu_mul_fp8_kernel<T, false>), grid, dim3(256), 0, st, (const T*)h,
                       h_stride, jobs, inter, groups, q, scales);
}

bool aligned(const void* p, int64_t stride, int elem) {
  return (uintptr_t)p % 16 == 0 && stride * elem % 16 == 0;
}

int refuse(int rc, const char* why, const char* where) {
  wisp_set_last_error(why, where);
  return rc;
}

}  // namespace
}  // namespace wisp

extern "C" int wisp_add_rms_norm(const void* x, int dtype, int64_t rows, int cols,
                                 int64_t x_stride, const void* residual, int residual_dtype,
                                 int64_t residual_stride, void* residual_out,
                                 int64_t residual_out_stride, const void* weight,
                                 int weight_dtype, float eps, void* out, uint8_t* q,
                                 float* scales, wisp_stream_t stream) {
  using namespace wisp;
  const char* where = "wisp_add_rms_norm";
  if (rows < 0 || cols < 0) return refuse(WISP_ERR_INVALID, "invalid matrix", where);
  if (rows == 0 || cols == 0) return WISP_OK;
  if (!x || !weight || (!out && !q) || (q && !scales) || (residual && !residual_out))
    return refuse(WISP_ERR_INVALID, "a buffer is missing", where);
  const bool bf16 = dtype == WISP_BF16;
  if ((!bf16 && dtype != WISP_F32) ||
      (weight_dtype != dtype && weight_dtype != WISP_F32) ||
      (residual && residual_dtype != dtype && residual_dtype != WISP_F32))
    return refuse(WISP_ERR_UNSUPPORTED, "x is float32 or bfloat16, weight and residual are of "
                  "its type or float32", where);
  if (cols > kMaxCols) return refuse(WISP_ERR_UNSUPPORTED, "more than 32768 columns", where);
  const bool wf = weight_dtype == WISP_F32, rf = residual_dtype == WISP_F32;
  const int xs = bf16 ? 2 : 4, rs = rf ? 4 : 2;
  const bool vec = cols % kPer == 0 && aligned(x, x_stride, xs) && aligned(weight, 0, 1) &&
                   (!residual || (aligned(residual, residual_stride, rs) &&
                                  aligned(residual_out, residual_out_stride, rs))) &&
                   (uintptr_t)out % 16 == 0 && (uintptr_t)q % 8 == 0;
  const NormArgs a = {x, residual, weight, residual_out, out, q, scales, rows, x_stride,
                      residual_stride, residual_out_stride, cols, (cols + kGroup - 1) / kGroup,
                      eps};
  hipStream_t st = (hipStream_t)stream;
  if (!bf16)
    return residual ? norm_of<float, float, float>(a, vec, st)
                    : norm_of<float, void, float>(a, vec, st);
  if (!residual)
    return wf ? norm_of<uint16_t, void, float>(a, vec, st)
              : norm_of<uint16_t, void, uint16_t>(a, vec, st);
  if (rf)
    return wf ? norm_of<uint16_t, float, float>(a, vec, st)
              : norm_of<uint16_t, float, uint16_t>(a, vec, st);
  return wf ? norm_of<uint16_t, uint16_t, float>(a, vec, st)
            : norm_of<uint16_t, uint16_t, uint16_t>(a, vec, st);
}

extern "C" int wisp_silu_mul_fp8(const void* h, int dtype, int64_t rows, int inter,
                                 int64_t h_stride, uint8_t* q, float* scales,
                                 wisp_stream_t stream) {
  using namespace wisp;
  const char* where = "wisp_silu_mul_fp8";
  if (rows < 0 || inter < 0 || (dtype != WISP_F32 && dtype != WISP_BF16))
    return refuse(WISP_ERR_INVALID, "invalid matrix", where);
  if (rows == 0 || inter == 0) return WISP_OK;
  if (!h || !q || !scales) return refuse(WISP_ERR_INVALID, "a buffer is missing", where);
  const int groups = (inter - 1) / kGroup + 1;
  if (rows > (int64_t)0xffffff * 16 / groups)  // (a launch has fewer than 2^32 threads)
    return refuse(WISP_ERR_UNSUPPORTED, "too many rows", where);
  const int64_t jobs = rows * groups;
  const int elem = dtype == WISP_F32 ? 4 : 2;
  const bool vec = inter % kPer == 0 && aligned(h, h_stride, elem) && (uintptr_t)q % 8 == 0;
  if (dtype == WISP_BF16)
    launch_silu<uint16_t>(h, h_stride, jobs, inter, groups, q, scales, vec, (hipStream_t)stream);
  else
    launch_silu<float>(h, h_stride, jobs, inter, groups, q, scales, vec, (hipStream_t)stream);
  WISP_HIP_TRY(hipGetLastError());
  return WISP_OK;
}
