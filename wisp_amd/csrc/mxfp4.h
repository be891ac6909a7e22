// MXFP4 on gfx950: E2M1 codes (two to a byte, the earlier value in the low
// half) with one E8M0 scale byte s per block of 32 values of a row; a value is
// E2M1(code) * 2^(s - 127), s = 255 is NaN.
//
// The conversions are single instructions that take the scale as a float
// whose exponent field is s.  Checked on MI355X over every byte and scale
// (reading back) and every finite bf16 value (quantising): exact, rounded to
// nearest with ties to the even code, saturating at 6, subnormal results and
// scales included.  A value read back is exact in bf16 too: two significant
// bits, and no exponent below bf16's subnormals.
#pragma once

#include <math.h>

#include "common.h"

namespace wisp {
namespace mx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 32;        // values of one scale
constexpr int kBlockBytes = 16;   // their codes

// The number of experts that the pairs of T tokens spread over, on average.
inline double distinct(int T, int K, int nslots) {
  const double e = nslots > K ? nslots : K;
  return e * (1.0 - pow(1.0 - K / e, T));
}

// The bits of the conversions' scale operand for byte `q` (0..3) of a word of
// scale bytes.
__device__ inline uint32_t scale_of(uint32_t word, int q) {
  return ((word >> (8 * q)) & 0xffu) << 23;
}

// The eight bf16 values of a word of codes, two to a word: half an operand row
// of the matrix instruction.  (Operands are held as words: the compiler takes
// a bf16 vector that lives across a branch apart, value by value.)
__device__ __attribute__((always_inline)) inline u32x4 bf16_of(uint32_t codes, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
}

// acc + a (16 rows x 32 of k) . b (32 of k x 16 columns).
__device__ __attribute__((always_inline)) inline f32x4 mfma(const u32x4& a, const u32x4& b,
                                                            const f32x4& acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}

// The same values two and two, and as float32.
struct Pairs {
  bf16x2 p[4];
};
__device__ __attribute__((always_inline)) inline Pairs pairs_of(uint32_t codes, float scale) {
  return Pairs{{__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0),
                __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1),
                __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2),
                __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3)}};
}
__device__ __attribute__((always_inline)) inline void f32_of(uint32_t codes, float scale,
                                                             float (&f)[8]) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
  f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1];
  f[4] = c[0], f[5] = c[1], f[6] = d[0], f[7] = d[1];
}

// c + a[0] * b[0] + a[1] * b[1] in float32, b's two bf16 values in a word.
__device__ __attribute__((always_inline)) inline float dot2(bf16x2 a, uint32_t b, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(a, __builtin_bit_cast(bf16x2, b), c, false);
}

// A range of less than 2^31 bytes of device memory, read by 32-bit byte
// offsets (`off`, a lane's, plus `base`, the wave's, which lies in the range);
// a read at or past the range's end gives zeros and touches no memory.
#ifdef __HIP_DEVICE_COMPILE__
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __attribute__((always_inline)) inline Buffer buffer(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00027000);
}
__device__ __attribute__((always_inline)) inline u32x4 load16_nt(Buffer b, uint32_t off,
                                                                   uint32_t base) {
  // nt: each byte is read once
  return __builtin_amdgcn_raw_buffer_load_b128(b, (int)off, (int)base, 2);
}
__device__ __attribute__((always_inline)) inline u32x4 load16(Buffer b, uint32_t off,
                                                                uint32_t base) {
  return __builtin_amdgcn_raw_buffer_load_b128(b, (int)off, (int)base, 0);
}
__device__ __attribute__((always_inline)) inline u32x2 load8(Buffer b, uint32_t off) {
  return __builtin_amdgcn_raw_buffer_load_b64(b, (int)off, 0, 0);
}
__device__ __attribute__((always_inline)) inline uint32_t load4(Buffer b, uint32_t off) {
  return __builtin_amdgcn_raw_buffer_load_b32(b, (int)off, 0, 0);
}
#else  // the host pass does not know these builtins
struct Buffer {};
__device__ inline Buffer buffer(const void*, uint32_t) { return {}; }
__device__ inline u32x4 load16_nt(Buffer, uint32_t, uint32_t) { return {}; }
__device__ inline u32x4 load16(Buffer, uint32_t, uint32_t) { return {}; }
__device__ inline u32x2 load8(Buffer, uint32_t) { return {}; }
__device__ inline uint32_t load4(Buffer, uint32_t) { return 0; }
#endif
}  // namespace mx
}  // namespace wisp
