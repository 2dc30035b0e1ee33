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
// Layout, of rows and of packed weights alike: 16 rows and 128 k are a tile of 2048 bytes, two planes of
// 64 k, in each 16 bytes for every one of 64 lanes: lane 16 g + r holds row r's k 16 g .. 16 g + 15. A
// wave's load is 1 KB in one piece; from rows that lie one behind the other it takes 64 bytes of each of
// 16, twice the lines for the address unit, which bounded the products (8192^3: 429 us, so 392). Scales
// are (kp / 32, mp) bytes, mp the rows rounded up to 128: of 128 rows, row 32 j + c's byte is the 4 c + j-th, so
// that a lane's four row tiles are one dword, of which the instruction's own selector picks a byte.
// Nothing is written for rows behind the last, or read from there into a result.
#pragma once

#include "m3s_common.h"

namespace m3s {

constexpr int kBlock8 = 32;    // values to a scale
constexpr int kStep8 = 128;    // K of one v_mfma_scale_f32_16x16x128_f8f6f4

__host__ __device__ inline int64_t padded_rows(int64_t rows) { return (rows + 127) & ~(int64_t)127; }
inline int64_t padded8(int64_t width) { return (width + kStep8 - 1) / kStep8 * kStep8; }

// Where row r's scales stand in a block's, and the byte of its k (a multiple of 8: 8 bytes lie together)
__device__ __forceinline__ int64_t scale_at(int64_t r) {
  return (r & ~(int64_t)127) + 4 * (r & 31) + ((r >> 5) & 3);
}
__device__ __forceinline__ int64_t value_at(int64_t r, int k, int steps) {
  return ((r >> 4) * steps + (k >> 7)) * 2048 + ((k >> 6) & 1) * 1024 + (((k >> 4) & 3) * 16 + (r & 15)) * 16 + (k & 15);
}

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
