// Rows to 8 bits on gfx950, alone or behind the block norm of the residual stream, and back.
//
//   s = x + add (rounded to the stream's type),  n = s / sqrt(mean_j s^2 + eps) gain,
//   rows in 8 bits of n (or of x, without a norm): m3s_eight.h has their form.
//
// The norm is m3s_rms_fwd's (rms_norm, layer.py:190-198, with the residual add of model.py:222-228)
// with another output; the statistics are float32 and n is never rounded to bf16 in between.
//
// HBM-bound: x and add in, s and the rows out, each once. A lane holds 8 neighbouring columns (one
// or two 16-byte loads, one 8-byte store), so a block's 32 are four lanes of a quad and its maximum
// is two DPP steps. A row stays in registers between its sum of squares and its rounding. A
// workgroup of 16 waves takes the 16 rows of a tile, so that their 16-byte pieces meet in one L2.
#include "m3s_eight.h"
#include "m3s_internal.h"

namespace m3s {

constexpr int kR8Waves = 16;
constexpr int kR8Threads = 64 * kR8Waves;
constexpr int kR8Pass = 64 * 8;                 // columns a wave takes at once
constexpr int kR8MaxWidth = kR8Waves * kR8Pass * 2;   // 16384, of a norm

struct R8Params {
  const void* x;
  const void* add;
  const float* gain;
  void* sum;
  uint8_t* values;
  uint8_t* scales;
  int64_t M, mp, ldx, lda;
  int D, kp, steps;
  float eps;
};

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int left, float (&v)[8]) {
  if constexpr (VEC) {
    if (left > 0) {
      if constexpr (sizeof(T) == 4) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
      } else {
        const bf16x8 a = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? (float)p[i] : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int left, const float (&v)[8]) {
  if constexpr (VEC) {
    if (left <= 0) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      bf16x8 a;
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = (bf16)v[i];
      *reinterpret_cast<bf16x8*>(p) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (T)v[i];
  }
}

__device__ __forceinline__ uint32_t quad_max(uint32_t u) {
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0xB1, 0xf, 0xf, true);   // xor 1
  u = u > o ? u : o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x4E, 0xf, 0xf, true);            // xor 2
  return u > o ? u : o;
}

// RW waves to a row (1, 4, 8 or 16), NP pieces of 8 columns to a lane, W columns together; without a norm RW is 1
// and the grid's second axis takes the columns. TURN: the tile's bytes and scales meet in LDS and go out in
// whole pieces; else (rows past 8192 columns) a lane's 8 bytes go where they belong (16384 x 2048 bf16: 30 us
// so, 24 turned). Rows that do not keep 16-byte boundaries are read a column to a lane, and each lane's 8
// columns come from LDS.
template <typename TX, bool NORM, bool ADD, bool VEC, int RW, int NP, bool TURN>
__global__ void __launch_bounds__(kR8Threads) rows8_kernel(const R8Params p) {
  constexpr int STEP = kR8Pass * RW, W = STEP * NP, LD = W + 16;
  __shared__ __attribute__((aligned(16))) uint8_t turn[TURN ? 16 * LD : 16];
  __shared__ uint8_t turn_scales[TURN ? W / 2 : 1];   // [block][row]
  __shared__ __attribute__((aligned(16))) float cols[VEC ? 4 : kR8Waves * kR8Pass];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int w0 = NORM ? 0 : (int)blockIdx.y * W, c0 = w0 + 8 * lane + kR8Pass * (wave % RW);
  const int64_t r0 = (int64_t)blockIdx.x * 16;
#pragma unroll 1
  for (int it = 0; it < RW; ++it) {
    const int rt = it * (kR8Waves / RW) + wave / RW;   // row of the tile
    const int64_t r = r0 + rt;
    const int D = r < p.M ? p.D : 0;
    const TX* xr = static_cast<const TX*>(p.x) + r * p.ldx;
    const bf16* ar = ADD ? static_cast<const bf16*>(p.add) + r * p.lda : nullptr;
    TX* sr = ADD ? static_cast<TX*>(p.sum) + r * p.D : nullptr;
    float v[NP][8];
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < NP; ++k) load8<TX, true>(xr + c0 + k * STEP, D - c0 - k * STEP, v[k]);
      if constexpr (ADD) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
          float d[8];
          load8<bf16, true>(ar + c0 + k * STEP, D - c0 - k * STEP, d);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[k][i] = (float)(TX)(v[k][i] + d[i]);
        }
#pragma unroll
        for (int k = 0; k < NP; ++k) store8<TX, true>(sr + c0 + k * STEP, D - c0 - k * STEP, v[k]);
      }
    } else {
      float* mine = cols + wave * kR8Pass;
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int c = c0 - 8 * lane + k * STEP + lane;
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = c + 64 * i < D ? (float)xr[c + 64 * i] : 0.f;
        if constexpr (ADD) {
          float d[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] = c + 64 * i < D ? (float)ar[c + 64 * i] : 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const TX sum = (TX)(t[i] + d[i]);
            t[i] = (float)sum;
            if (c + 64 * i < D) sr[c + 64 * i] = sum;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[lane + 64 * i] = t[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const f32x4 a = *reinterpret_cast<const f32x4*>(mine + 8 * lane), b = *reinterpret_cast<const f32x4*>(mine + 8 * lane + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[k][i] = a[i]; v[k][4 + i] = b[i]; }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < NP; ++k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += v[k][i] * v[k][i];
      }
      ss = wave_total(ss);
      if constexpr (RW > 1) {
        __shared__ float part[2][kR8Waves];   // by turns: one barrier a row
        if (lane == 0) part[it & 1][wave] = ss;
        __syncthreads();
        ss = 0.f;
#pragma unroll
        for (int w = 0; w < RW; ++w) ss += part[it & 1][wave / RW * RW + w];
      }
      const float rs = 1.f / sqrtf(ss / (float)p.D + p.eps);
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        float g[8];
        const int c = c0 + k * STEP;
        if (VEC || c + 8 <= p.D) load8<float, true>(p.gain + c, p.D - c, g);   // gain is on its boundary
        else load8<float, false>(p.gain + c, p.D - c, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k][i] = v[k][i] * rs * g[i];
      }
    }
    // a column behind the width is a zero, whatever the row's statistics are (zero times the inverse
    // of a NaN is not)
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int c = c0 + k * STEP;
      if (c >= p.kp || r >= p.M) continue;   // whole quads: kp is a multiple of 128
      if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i >= p.D) v[k][i] = 0.f;
      }
      uint32_t u = quad_max(max_bits(v[k]));
      if (u >= kInfBits) u = quad_max(max_bits_finite(v[k]));   // a quad takes this together
      const int byte = scale_byte(u);
      const float down = scale_down(byte);
      const i32x2_ q = {pack4(v[k][0], v[k][1], v[k][2], v[k][3], down),
                        pack4(v[k][4], v[k][5], v[k][6], v[k][7], down)};
      if constexpr (TURN) {
        *reinterpret_cast<i32x2_*>(turn + rt * LD + c - w0) = q;
        if ((lane & 3) == 0) turn_scales[(c - w0) / 2 + rt] = (uint8_t)byte;
      } else {
        *reinterpret_cast<i32x2_*>(p.values + value_at(r, c, p.steps)) = q;
        if ((lane & 3) == 0) p.scales[(int64_t)(c / kBlock8) * p.mp + scale_at(r)] = (uint8_t)byte;
      }
    }
  }
  if constexpr (TURN) {
    __syncthreads();
    const int n = min(W, p.kp - w0);   // the window's columns, and its tile's pieces of 16 bytes
    const int rows = (int)min(p.M - r0, (int64_t)16);
    uint8_t* out = p.values + (int64_t)blockIdx.x * p.steps * 2048 + w0 * 16;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int row = i & 15;
      if (row < rows)
        *reinterpret_cast<i32x4_*>(out + 16 * i) =
            *reinterpret_cast<const i32x4_*>(turn + row * LD + (i >> 7) * 128 + ((i >> 4) & 7) * 16);
    }
    for (int i = threadIdx.x; i < n / 2; i += blockDim.x) {
      const int row = i & 15;
      if (row < rows)
        p.scales[(int64_t)(w0 / kBlock8 + (i >> 4)) * p.mp + scale_at(r0 + row)] = turn_scales[i];
    }
  }
}

// 8 columns to a lane: the values that the bytes stand for
template <typename TY, bool VEC>
__global__ void __launch_bounds__(kR8Threads) rows8_values_kernel(const uint8_t* __restrict__ values,
                                                                  const uint8_t* __restrict__ scales,
                                                                  TY* __restrict__ y, int64_t M, int D,
                                                                  int steps) {
  __shared__ __attribute__((aligned(16))) float cols[VEC ? 4 : kR8Waves * kR8Pass];   // a row's, to leave a column a lane
  const int64_t r = (int64_t)blockIdx.x * kR8Waves + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, w0 = (int)blockIdx.y * kR8Pass, c = 8 * lane + w0;
  if (r >= M) return;   // whole waves
  float v[8] = {};
  if (c < D) {
    const i32x2_ q = *reinterpret_cast<const i32x2_*>(values + value_at(r, c, steps));
    const float up = scale_up(scales[(int64_t)(c / kBlock8) * padded_rows(M) + scale_at(r)]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(q[h], false);
      const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(q[h], true);
      v[4 * h] = lo[0] * up; v[4 * h + 1] = lo[1] * up;
      v[4 * h + 2] = hi[0] * up; v[4 * h + 3] = hi[1] * up;
    }
  }
  if constexpr (VEC) {
    store8<TY, true>(y + r * D + c, D - c, v);
  } else {
    float* mine = cols + (threadIdx.x >> 6) * kR8Pass;
    *reinterpret_cast<f32x4*>(mine + 8 * lane) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(mine + 8 * lane + 4) = f32x4{v[4], v[5], v[6], v[7]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = w0 + lane + 64 * i;
      if (at < D) y[r * D + at] = (TY)mine[lane + 64 * i];
    }
  }
}

template <typename TX, bool NORM, bool ADD, bool VEC>
static void launch_rows8(const R8Params& p, hipStream_t s) {
  const unsigned tiles = (unsigned)((p.M + 15) / 16);
  const unsigned few = 64 * (unsigned)(p.M < 16 ? p.M : 16);   // a wave to a row, and none for rows that are not there
#define M3S_R8(RW, NP, TURN, GRID, THREADS) \
  hipLaunchKernelGGL((rows8_kernel<TX, NORM, ADD, VEC, RW, NP, TURN>), GRID, dim3(THREADS), 0, s, p)
  // Fewer rows than a tile has nothing to turn (1 x 768: 3.4 us, so 2.1). Several waves to a row leave each fewer
  // registers, and a CU two workgroups (16384 x 2048 bf16: one wave a row 34 us, four 29).
  if constexpr (!NORM) {
    const dim3 grid(tiles, (unsigned)((p.kp + 2 * kR8Pass - 1) / (2 * kR8Pass)));
    if (p.M < 16) M3S_R8(1, 2, false, grid, few);
    else if (p.kp <= kR8Pass) M3S_R8(1, 1, true, grid, few);
    else M3S_R8(1, 2, true, grid, few);
  } else {
    const int pieces = (p.kp + kR8Pass - 1) / kR8Pass;
    if (p.M < 16 && pieces <= 2) M3S_R8(1, 2, false, dim3(tiles), few);
    else if (pieces <= 1) M3S_R8(1, 1, true, dim3(tiles), few);
    else if (pieces <= 2) M3S_R8(1, 2, true, dim3(tiles), few);
    else if (pieces <= 4) M3S_R8(4, 1, true, dim3(tiles), kR8Threads);
    else if (pieces <= 8) M3S_R8(8, 1, true, dim3(tiles), kR8Threads);
    else if (pieces <= 16) M3S_R8(16, 1, VEC, dim3(tiles), kR8Threads);   // LDS holds no columns besides
    else M3S_R8(16, 2, false, dim3(tiles), kR8Threads);
  }
#undef M3S_R8
}

template <bool NORM, bool ADD>
static void dispatch_rows8(const m3s_rows8_args* a, const R8Params& p, hipStream_t s) {
  const int xs = a->x_dtype == M3S_DTYPE_BF16 ? 2 : 4;
  // 8 columns at once where rows and pointers keep them on their boundary
  const bool vec = p.D % 8 == 0 && p.ldx % 8 == 0 && (uintptr_t)p.x % 16 == 0 &&
                   (!ADD || (p.lda % 8 == 0 && (uintptr_t)p.add % 16 == 0 && (uintptr_t)p.sum % 16 == 0));
  if (xs == 2) vec ? launch_rows8<bf16, NORM, ADD, true>(p, s) : launch_rows8<bf16, NORM, ADD, false>(p, s);
  else vec ? launch_rows8<float, NORM, ADD, true>(p, s) : launch_rows8<float, NORM, ADD, false>(p, s);
}

}  // namespace m3s

using namespace m3s;

extern "C" int32_t m3s_rows8(const m3s_rows8_args* a, void* stream) {
  clear_error();
  M3S_REQUIRE(a != nullptr, "m3s_rows8: args is NULL");
  M3S_REQUIRE(a->struct_size == (int32_t)sizeof(m3s_rows8_args),
              "m3s_rows8: struct_size %d != %d (ABI mismatch)", a->struct_size,
              (int)sizeof(m3s_rows8_args));
  M3S_REQUIRE(a->x_dtype == M3S_DTYPE_BF16 || a->x_dtype == M3S_DTYPE_F32, "m3s_rows8: bad x_dtype %d",
              a->x_dtype);
  M3S_REQUIRE(a->rows >= 0 && a->rows <= M3S_ROWS8_MAX && a->width > 0 && a->width <= M3S_ROWS8_WIDTH_MAX,
              "m3s_rows8: rows %lld or width %d out of range", (long long)a->rows, a->width);
  M3S_REQUIRE(!a->gain || a->width <= kR8MaxWidth, "m3s_rows8: width %d of a norm is over %d", a->width,
              kR8MaxWidth);
  if (a->rows == 0) return 0;
  M3S_REQUIRE(a->x && a->values && a->scales, "m3s_rows8: NULL pointer");
  M3S_REQUIRE((a->add == nullptr) == (a->sum == nullptr) && (!a->add || a->gain),
              "m3s_rows8: give both add and sum, with a gain, or neither");
  M3S_REQUIRE(a->ldx >= a->width && (!a->add || a->ldadd >= a->width), "m3s_rows8: a row stride is too short");
  M3S_REQUIRE((uintptr_t)a->values % 16 == 0 && (uintptr_t)a->gain % 16 == 0,
              "m3s_rows8: values and gain must be 16-byte aligned");
  R8Params p{a->x, a->add, a->gain, a->sum, static_cast<uint8_t*>(a->values),
             static_cast<uint8_t*>(a->scales), a->rows, padded_rows(a->rows), a->ldx, a->ldadd, a->width,
             (int)padded8(a->width), (int)(padded8(a->width) / kStep8), a->eps};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!a->gain) dispatch_rows8<false, false>(a, p, s);
  else if (!a->add) dispatch_rows8<true, false>(a, p, s);
  else dispatch_rows8<true, true>(a, p, s);
  return launch_status("m3s_rows8");
}

extern "C" int32_t m3s_rows8_values(const m3s_rows8_values_args* a, void* stream) {
  clear_error();
  M3S_REQUIRE(a != nullptr, "m3s_rows8_values: args is NULL");
  M3S_REQUIRE(a->struct_size == (int32_t)sizeof(m3s_rows8_values_args),
              "m3s_rows8_values: struct_size %d != %d (ABI mismatch)", a->struct_size,
              (int)sizeof(m3s_rows8_values_args));
  M3S_REQUIRE(a->y_dtype == M3S_DTYPE_BF16 || a->y_dtype == M3S_DTYPE_F32,
              "m3s_rows8_values: bad y_dtype %d", a->y_dtype);
  M3S_REQUIRE(a->rows >= 0 && a->rows <= M3S_ROWS8_MAX && a->width > 0 && a->width <= M3S_ROWS8_WIDTH_MAX,
              "m3s_rows8_values: rows %lld or width %d out of range", (long long)a->rows, a->width);
  if (a->rows == 0) return 0;
  M3S_REQUIRE(a->values && a->scales && a->y, "m3s_rows8_values: NULL pointer");
  M3S_REQUIRE((uintptr_t)a->values % 16 == 0, "m3s_rows8_values: values must be 16-byte aligned");
  const int kp = (int)padded8(a->width);
  const dim3 grid((unsigned)((a->rows + kR8Waves - 1) / kR8Waves), (unsigned)((kp + kR8Pass - 1) / kR8Pass));
  const uint8_t *v = static_cast<const uint8_t*>(a->values), *c = static_cast<const uint8_t*>(a->scales);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool vec = a->width % 8 == 0 && (uintptr_t)a->y % 16 == 0;
#define M3S_R8V(TY, VEC)                                                                          \
  hipLaunchKernelGGL((rows8_values_kernel<TY, VEC>), grid, dim3(kR8Threads), 0, s, v, c,          \
                     static_cast<TY*>(a->y), a->rows, a->width, kp / kStep8)
  if (a->y_dtype == M3S_DTYPE_BF16) {
    if (vec) M3S_R8V(bf16, true);
    else M3S_R8V(bf16, false);
  } else {
    if (vec) M3S_R8V(float, true);
    else M3S_R8V(float, false);
  }
#undef M3S_R8V
  return launch_status("m3s_rows8_values");
}
