// Rows in 8 bits, as the matrix cores' block-scaled products take them: e4m3 values in blocks of
// 32 along the summed axis, each block with a scale 2^e, e + 127 held in a byte.
//
//   e = the smallest integer >= -126 with max_i |x_i| 2^-e <= 448 (e4m3's largest value),
//   q_i = x_i 2^-e to the nearest e4m3 (ties to even).
//
// Nothing saturates: with the binade of the maximum as the exponent (e4m3's largest binade ends at
// 480) a maximum above 448 would lose up to 6.7% of itself. Multiplying by 2^-e is exact but for
// results below 2^-126, far under e4m3's smallest step, so each value is rounded once. A
// non-finite entry becomes e4m3's NaN and does not count for the maximum: its row's products are
// NaN, as they would be in floating point, and its block's other values keep their scale.
//
// Layout: values (rows, kp) bytes with kp the width rounded up to 128 (zeros behind the width), the
// K of one matrix instruction, and scales (kp / 32, mp) bytes with mp the rows rounded up to 16: a
// block's scales of four rows are one dword, which the products' lanes read at once and pick
// their byte of by the instruction's own selector. Nothing writes the scales behind the last row.
#pragma once

#include "m3s_common.h"

namespace m3s {

constexpr int kBlock8 = 32;    // values to a scale
constexpr int kStep8 = 128;    // K of one v_mfma_scale_f32_16x16x128_f8f6f4

__host__ __device__ inline int64_t padded16(int64_t rows) { return (rows + 15) & ~(int64_t)15; }
inline int64_t padded8(int64_t width) { return (width + kStep8 - 1) / kStep8 * kStep8; }

typedef int i32x2_ __attribute__((ext_vector_type(2)));
typedef int i32x4_ __attribute__((ext_vector_type(4)));
typedef int i32x8_ __attribute__((ext_vector_type(8)));

constexpr uint32_t kInfBits = 0x7f800000u;

__device__ __forceinline__ uint32_t abs_bits(float v) {
  return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
}
// The largest magnitude's bits, which order as the magnitudes do; NaN is passed over, an infinity
// comes out as kInfBits.
template <int N>
__device__ __forceinline__ uint32_t max_bits(const float (&v)[N]) {
  float u = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) u = __builtin_fmaxf(u, __builtin_fabsf(v[i]));
  return __builtin_bit_cast(uint32_t, u);
}
// ... of the finite entries alone
template <int N>
__device__ __forceinline__ uint32_t max_bits_finite(const float (&v)[N]) {
  uint32_t u = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t b = abs_bits(v[i]);
    if (b < kInfBits && b > u) u = b;
  }
  return u;
}

// The scale byte of a block whose maximum has these bits: its exponent field less 8, one more where
// its mantissa is above 448's (1.75).
__device__ __forceinline__ int scale_byte(uint32_t u) {
  const int e = (int)((u + 0x1fffffu) >> 23) - 8;
  return e > 1 ? e : 1;
}
__device__ __forceinline__ float scale_down(int byte) {   // 2^-e
  return __builtin_bit_cast(float, (uint32_t)(254 - byte) << 23);
}
__device__ __forceinline__ float scale_up(int byte) {     // 2^e
  return __builtin_bit_cast(float, (uint32_t)byte << 23);
}

// four values times 2^-e, as four bytes
__device__ __forceinline__ int pack4(float a, float b, float c, float d, float down) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a * down, b * down, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c * down, d * down, r, true);
}

}  // namespace m3s
