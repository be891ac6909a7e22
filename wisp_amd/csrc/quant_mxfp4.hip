// Quantising rows to MXFP4 and reading them back (format: mxfp4.h).
//
// Per block of 32 values of a row, m = max|v|:
//   s = clamp(floor(log2 m) - 2, -127, 127)      (m = 0: -127)
//   code = E2M1(v / 2^s), nearest, ties to the even code, saturating at 6
// so that the largest value of a block lands in [4, 8).  A block that holds
// an infinity or a NaN gets scale byte 255 and zero codes: it reads back as
// NaNs.  Rows are whole blocks and contiguous, so a matrix is one run of
// blocks whatever its shape.
//
// Both are streams: a lane holds eight values, one word of codes, and four
// lanes hold a block, so that every load and store of a wave is one
// contiguous run (16 bytes of bf16 or two times 16 of float32 a lane); a thread
// has four words' loads in flight.  Bound by memory.  Measured, bf16: 24576 x
// 2048 values quantised in 24.3 us (5.2 TB/s of values, codes and scales) and
// read back in 19.7 us (6.5 TB/s), 28672 x 4096 read back in 48 us (6.2 TB/s).
#include "mxfp4.h"

namespace wisp {
namespace {

constexpr int kPer = 8;     // values a lane
constexpr int kAtOnce = 4;  // words of codes a thread has in flight

// Eight consecutive values as float32.
__device__ inline void load8(const uint16_t* p, float (&v)[kPer]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}
__device__ inline void load8(const float* p, float (&v)[kPer]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// words: 4 a block, so the four lanes of a block are in range together.
template <typename T>
__global__ __launch_bounds__(256) void quant_mxfp4_kernel(const T* __restrict__ x, int64_t words,
                                                          uint32_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
  const int64_t first = (int64_t)blockIdx.x * (256 * kAtOnce) + threadIdx.x;
  float v[kAtOnce][kPer];
#pragma unroll
  for (int n = 0; n < kAtOnce; ++n)
    if (first + n * 256 < words) load8(x + (first + n * 256) * kPer, v[n]);
#pragma unroll
  for (int n = 0; n < kAtOnce; ++n) {
    const int64_t i = first + n * 256;
    if (i >= words) continue;
    // magnitudes compare as their bits; an infinity or NaN is at least 255 << 23
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) m = max(m, __float_as_uint(v[n][j]) & 0x7fffffffu);
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, false));  // xor 1
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, false));  // xor 2
    const uint32_t e = m >> 23;
    const uint32_t s = e == 255 ? 255u : e < 2 ? 0u : e - 2;
    const float scale = __uint_as_float(s << 23);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[n][0], v[n][1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[n][2], v[n][3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[n][4], v[n][5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[n][6], v[n][7], scale, 3);
    codes[i] = s == 255 ? 0u : w;
    if ((i & 3) == 0) scales[i >> 2] = (uint8_t)s;
  }
}

__device__ inline void store8(uint16_t* p, uint32_t codes, float scale) {
  *reinterpret_cast<mx::u32x4*>(p) = mx::bf16_of(codes, scale);
}
__device__ inline void store8(float* p, uint32_t codes, float scale) {
  const mx::f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
  const mx::f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
  const mx::f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
  const mx::f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
  reinterpret_cast<float4*>(p)[0] = make_float4(a[0], a[1], b[0], b[1]);
  reinterpret_cast<float4*>(p)[1] = make_float4(c[0], c[1], d[0], d[1]);
}

template <typename T>
__global__ __launch_bounds__(256) void dequant_mxfp4_kernel(const uint32_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales,
                                                            int64_t words, T* __restrict__ out) {
  const int64_t first = (int64_t)blockIdx.x * (256 * kAtOnce) + threadIdx.x;
  uint32_t w[kAtOnce], s[kAtOnce];
#pragma unroll
  for (int n = 0; n < kAtOnce; ++n) {
    const int64_t i = first + n * 256;
    if (i < words) w[n] = codes[i], s[n] = scales[i >> 2];
  }
#pragma unroll
  for (int n = 0; n < kAtOnce; ++n) {
    const int64_t i = first + n * 256;
    if (i < words) store8(out + i * kPer, w[n], __uint_as_float(s[n] << 23));
  }
}

// What both entry points check; *words: the run's words of codes.
int check(const void* wide, int dtype, int64_t rows, int cols, const void* codes,
          const void* scales, int64_t* words, const char* where) {
  *words = 0;
  if (rows < 0 || cols < 0 || (dtype != WISP_F32 && dtype != WISP_BF16) ||
      (rows > 0 && cols > 0 && (!wide || !codes || !scales))) {
    wisp_set_last_error("invalid matrix", where);
    return WISP_ERR_INVALID;
  }
  if (cols % mx::kBlock || ((uintptr_t)wide) % 16 || ((uintptr_t)codes) % 4) {
    wisp_set_last_error("cols must be a multiple of 32, values 16-byte and codes 4-byte aligned",
                        where);
    return WISP_ERR_UNSUPPORTED;
  }
  // (a launch has fewer than 2^32 threads)
  if (cols > 0 && rows > (int64_t)0xffffff * (256 * kAtOnce) / (cols / kPer)) {
    wisp_set_last_error("matrix too large", where);
    return WISP_ERR_UNSUPPORTED;
  }
  *words = rows * (cols / kPer);
  return WISP_OK;
}

dim3 grid_of(int64_t words) { return dim3((unsigned)((words + 256 * kAtOnce - 1) / (256 * kAtOnce))); }

}  // namespace
}  // namespace wisp

extern "C" int wisp_quant_mxfp4(const void* x, int dtype, int64_t rows, int cols, uint8_t* codes,
                                uint8_t* scales, wisp_stream_t stream) {
  using namespace wisp;
  int64_t words;
  const int rc = check(x, dtype, rows, cols, codes, scales, &words, "wisp_quant_mxfp4");
  if (rc != WISP_OK || words == 0) return rc;
  if (dtype == WISP_BF16)
    hipLaunchKernelGGL(quant_mxfp4_kernel<uint16_t>, grid_of(words), dim3(256), 0,
                       (hipStream_t)stream, (const uint16_t*)x, words, (uint32_t*)codes, scales);
  else
    hipLaunchKernelGGL(quant_mxfp4_kernel<float>, grid_of(words), dim3(256), 0,
                       (hipStream_t)stream, (const float*)x, words, (uint32_t*)codes, scales);
  WISP_HIP_TRY(hipGetLastError());
  return WISP_OK;
}

extern "C" int wisp_dequant_mxfp4(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                  int cols, void* out, int dtype, wisp_stream_t stream) {
  using namespace wisp;
  int64_t words;
  const int rc = check(out, dtype, rows, cols, codes, scales, &words, "wisp_dequant_mxfp4");
  if (rc != WISP_OK || words == 0) return rc;
  if (dtype == WISP_BF16)
    hipLaunchKernelGGL(dequant_mxfp4_kernel<uint16_t>, grid_of(words), dim3(256), 0,
                       (hipStream_t)stream, (const uint32_t*)codes, scales, words, (uint16_t*)out);
  else
    hipLaunchKernelGGL(dequant_mxfp4_kernel<float>, grid_of(words), dim3(256), 0,
                       (hipStream_t)stream, (const uint32_t*)codes, scales, words, (float*)out);
  WISP_HIP_TRY(hipGetLastError());
  return WISP_OK;
}
