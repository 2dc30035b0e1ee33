// Products of rows and weights in 8 bits on gfx950 (m3s_eight.h), with bias, activation and residual,
// or the MLP's gate and its rows in 8 bits again, in the epilogue:
//
//   y = act(x w + bias) + residual                    in bf16
//   a = value silu(gate), value | gate = x w + bias   in 8 bits, the next product's rows
//
// They stand for the projections of the LM (layer.py:233, 256; model.py:125-140, 231) on weights in
// 8 bits.
//
// Rows are the B operand and the weight A, so a lane's accumulators are neighbouring outputs of one row.
// There are two ways to a sum, chosen by whoever packs the weight:
//
// Float32 (the default): e4m3 values and their scales widen to bf16, which holds them (widen8), and
// v_mfma_f32_*_bf16 multiplies them: 4e-8 of a product of N(0, 1) rows, as float32 in any order.
//
// Short: v_mfma_scale_f32_*_f8f6f4 multiplies the 8 bits themselves, at twice bf16's rate, and applies a
// scale for every 32 of them on the way. Of each 8 neighbouring products it cuts what is below 2^-13 of the
// largest one's power of two, and adds the rest to the float32 accumulator (found with pairs of products;
// groups of 8 do not touch each other). A product of N(0, 1) rows is 1.3e-5 off for any K from 1024 to
// 16384; where large products cancel, small ones beside them are gone. What layouts and stores measure
// below was measured with short sums, where it weighs most.
//
// Weights are packed once (eightbit.pack8) in the rows' own tiles, their outputs being the rows. Four
// tiles are a group of 64 outputs: tile t, row 4 g + i is output 64 grp + 32 (t >> 1) + 8 g +
// 4 (t & 1) + i, which leaves a lane 8 neighbouring outputs (16 bytes of bf16) in two tiles, and four
// lanes the 32 of a block. With a gate, tiles 0 and 1 hold value's outputs 32 grp + 8 g + 4 t + i and
// tiles 2 and 3 gate's, so a lane has both.
#include <type_traits>

#include "m3s_eight.h"
#include "m3s_internal.h"
#include "m3s_tiles8.h"

namespace m3s {

enum Act8 { kActNone = M3S_ACT_NONE, kActSilu = M3S_ACT_SILU, kActGelu = M3S_ACT_GELU, kActRelu = M3S_ACT_RELU };

struct M8Params {
  const void* x;           // packed tiles, or (M, K) bf16 / float32 for few rows
  const uint8_t* xs;       // (4 KB, mp)
  const uint8_t* w;        // packed tiles
  const uint8_t* ws;       // [step][group of four tiles][lane][4]
  const float* bias;
  const bf16* residual;
  bf16* y;
  uint8_t* yv;             // gated: packed values and (4 steps, mp) scales
  uint8_t* ys;
  int64_t M, mp, ldx, ldr, ldy;
  int K, KB, N, NP, act, vec;   // N: outputs (half the weight's columns with a gate); NP: packed rows
  int tiles_m, tiles_n;
};

// v / (1 + e^-v) by the hardware's exponential and reciprocal, an ulp each (a division in full is some
// ten instructions of the gate's epilogue). e^-v past float32 is an infinity, and the result -0.
__device__ __forceinline__ float silu8(float v) {
  return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * v));
}
__device__ __forceinline__ float act8(float v, int act) {
  if (act == kActSilu) return silu8(v);
  // 1 + erf as erfc, which keeps its bits where the two cancel (at -5 the sum has four left)
  if (act == kActGelu) return 0.5f * v * erfcf(v * -0.70710678118654752f);
  if (act == kActRelu) return v > 0.f ? v : (v == v ? 0.f : v);
  return v;
}

__device__ __forceinline__ uint32_t max_lanes16(uint32_t u) {   // over the four lanes of a row
  uint32_t o = (uint32_t)__shfl_xor((int)u, 16, 64);
  u = u > o ? u : o;
  o = (uint32_t)__shfl_xor((int)u, 32, 64);
  return u > o ? u : o;
}

// 8 neighbouring outputs n .. n + 7 of row m.
__device__ __forceinline__ void finish8(const M8Params& p, int64_t m, int n, float (&v)[8]) {
  if (n >= p.N) return;
  const bool whole = (p.vec & 1) && n + 8 <= p.N;   // pointers and strides allow 16 bytes
  if (p.bias) {
    if (whole) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p.bias + n), b = *reinterpret_cast<const f32x4*>(p.bias + n + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[i] += a[i]; v[4 + i] += b[i]; }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < p.N) v[i] += p.bias[n + i];
    }
  }
  if (p.act != kActNone) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act8(v[i], p.act);
  }
  if (p.residual) {
    const bf16* rr = p.residual + m * p.ldr + n;
    if (whole) {
      const bf16x8 a = *reinterpret_cast<const bf16x8*>(rr);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += (float)a[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < p.N) v[i] += (float)rr[i];
    }
  }
  bf16* yr = p.y + m * p.ldy + n;
  if (whole) {
    bf16x8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (bf16)v[i];
    *reinterpret_cast<bf16x8*>(yr) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < p.N) yr[i] = (bf16)v[i];
  }
}

// A group's four accumulator tiles of row m. The gate's block of 32 outputs is the row's four lanes;
// outputs behind N are zeros (the packed weight has zero rows there), up to the rows' padded width.
template <bool GATED>
__device__ __forceinline__ void finish_group(const M8Params& p, int64_t m, int grp, int lane,
                                             const f32x4 (&acc)[4]) {
  const int g = lane >> 4;
  if constexpr (!GATED) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[i] = acc[2 * h][i]; v[4 + i] = acc[2 * h + 1][i]; }
      finish8(p, m, 64 * grp + 32 * h + 8 * g, v);
    }
  } else {
    const int j = 32 * grp + 8 * g;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float a = acc[i >> 2][i & 3], b = acc[2 + (i >> 2)][i & 3];
      if (p.bias) {
        const int c = min(j + i, p.N - 1);
        a += p.bias[c];
        b += p.bias[p.N + c];
      }
      v[i] = j + i < p.N ? a * silu8(b) : 0.f;
    }
    uint32_t u = max_lanes16(max_bits(v));
    if (u >= kInfBits) u = max_lanes16(max_bits_finite(v));
    const int byte = scale_byte(u);
    const float down = scale_down(byte);
    *reinterpret_cast<i32x2_*>(p.yv + value_at(m, j, p.NP / 256)) =
        i32x2_{pack4(v[0], v[1], v[2], v[3], down), pack4(v[4], v[5], v[6], v[7], down)};
    if (g == 0) p.ys[(int64_t)grp * p.mp + scale_at(m)] = (uint8_t)byte;
  }
}

// the wave's writes to LDS stand before its reads of what other lanes wrote (its LDS accesses
// complete in order; this keeps the compiler from moving one over the other)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ i32x8_ join8(i32x4_ a, i32x4_ b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// byte SA of sa and byte SB of sb are the operands' scales
template <int SA, int SB>
__device__ __forceinline__ void mma8(f32x4& acc, i32x8_ a, int sa, i32x8_ b, int sb) {
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, SA, sa, SB, sb);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F f) {
  if constexpr (N > 0) {
    static_for<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// ---- few rows ---------------------------------------------------------------------------
// The weight is the traffic. A workgroup takes a group of 64 outputs and 16 MT rows; its eight waves take the steps of
// K in turn, each loading its tiles straight to registers, and their sums meet in LDS in wave order
// (deterministic). The loads hide what float32 sums take more than short ones (1 x 1024 x 4480 3.6 us, short 3.4;
// 64 rows 4.4 and 4.0). Float rows are rounded to 8
// bits on the way in: a block is two lanes' half rows.
constexpr int kFewWaves = 8;
enum Rows8Kind { kRows8 = 0, kRowsBf16 = 1, kRowsF32 = 2 };

// A lane's share of rows m0 .. m0 + 15 of a step as memory holds it, so that nothing waits for its loads
// where they are issued: 8 bits and a scale, or floats in 16-byte pieces. Rows behind the last read the
// last one and give nothing but their own products, which are not stored.
template <int XK>
struct RowsRaw {
  i32x4_ v[XK == kRowsF32 ? 8 : 4];
};
template <>
struct RowsRaw<kRows8> {
  i32x8_ b;
  int sb;
};

template <int XK>
__device__ __forceinline__ void load_rows(const M8Params& p, int64_t m0, int kb, int lane, RowsRaw<XK>& x) {
  const int r = lane & 15, g = lane >> 4;
  if constexpr (XK == kRows8) {
    const int64_t tile = min(m0, p.M - 1) >> 4;
    const uint8_t* xr = static_cast<const uint8_t*>(p.x) + (tile * p.KB + kb) * 2048 + 16 * lane;
    x.b = join8(*reinterpret_cast<const i32x4_*>(xr), *reinterpret_cast<const i32x4_*>(xr + 1024));
    x.sb = p.xs[((int64_t)kb * 4 + g) * p.mp + scale_at(m0 + r)];
  } else {
    using TX = std::conditional_t<XK == kRowsBf16, bf16, float>;
    constexpr int E = 16 / sizeof(TX);   // a piece's
    const TX* xr = static_cast<const TX*>(p.x) + min(m0 + r, p.M - 1) * p.ldx;
    const int c0 = kb * kStep8 + 16 * g;
    if (p.vec & 2) {   // whole pieces; K % 8 == 0
#pragma unroll
      for (int i = 0; i < 32 / E; ++i) {
        const int c = c0 + 64 * (i / (16 / E)) + E * (i % (16 / E));
        x.v[i] = *reinterpret_cast<const i32x4_*>(xr + min(c, p.K - E));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32 / E; ++i) {
        const int c = c0 + 64 * (i / (16 / E)) + E * (i % (16 / E));
        TX t[E];
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = xr[min(c + e, p.K - 1)];
        x.v[i] = __builtin_bit_cast(i32x4_, t);
      }
    }
  }
}

// lane's operand and scale of them; `left` columns lie before the width's end
template <int XK>
__device__ __forceinline__ void rows_operand(const RowsRaw<XK>& x, int left, int lane, i32x8_& b, int& sb) {
  if constexpr (XK == kRows8) {
    b = x.b;
    sb = x.sb;
  } else {
    const int r = lane & 15, g = lane >> 4;
    int q[8], byte[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float f;
        if constexpr (XK == kRowsF32) f = __builtin_bit_cast(f32x4, x.v[4 * h + e / 4])[e % 4];
        else f = (float)__builtin_bit_cast(bf16x8, x.v[2 * h + e / 8])[e % 8];
        v[e] = 64 * h + 16 * g + e < left ? f : 0.f;
      }
      uint32_t u = max_bits(v), o = (uint32_t)__shfl_xor((int)u, 16, 64);
      u = u > o ? u : o;
      if (u >= kInfBits) {   // both lanes of the block
        u = max_bits_finite(v);
        o = (uint32_t)__shfl_xor((int)u, 16, 64);
        u = u > o ? u : o;
      }
      byte[h] = scale_byte(u);
      const float down = scale_down(byte[h]);
#pragma unroll
      for (int i = 0; i < 4; ++i) q[4 * h + i] = pack4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], down);
    }
    b = i32x8_{q[0], q[1], q[2], q[3], q[4], q[5], q[6], q[7]};
    // block g is half g >> 1 of the lanes 2 (g & 1), 2 (g & 1) + 1
    const int from = r + 32 * (g & 1);
    const int s0 = __shfl(byte[0], from, 64), s1 = __shfl(byte[1], from, 64);
    sb = g & 2 ? s1 : s0;
  }
}

// the scale of each plane's 16 bytes, from the lane that holds its block's
__device__ __forceinline__ int plane_scale(int s, int lane, int h) {
  return __shfl(s, (lane & 15) + 16 * (2 * h + (lane >> 5)), 64);
}
// Bytes 8 i .. 8 i + 7 of an operand, in bfloat16 with their scale 2^(byte - 127): exact from 2^-126 to below
// 2^128. 256 2^120 (float32's last values, 3.4e38) is an infinity, as it is where the rows are read back, and of
// values of a block of the least scale, below 2^-126, the bits under 2^-133 are lost.
__device__ __forceinline__ bf16x8 widen8(i32x8_ v, int i, int byte) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const float s = __int_as_float((byte & 255) << 23);
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * i], s, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * i], s, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * i + 1], s, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * i + 1], s, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <int MT, int XK, bool GATED, bool SHORT>
__global__ void __launch_bounds__(64 * kFewWaves) matmul8_few_kernel(const M8Params p) {
  constexpr int NT = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tile0 = blockIdx.x * NT;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  __shared__ __attribute__((aligned(16))) f32x4 part[kFewWaves][MT][NT][64];
  f32x4 acc[MT][NT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const uint8_t* wt = p.w + (int64_t)tile0 * p.KB * 2048 + 16 * lane;
  const uint8_t* st = p.ws + 64 * tile0 + 4 * lane;
  for (int kb = wave; kb < p.KB; kb += kFewWaves) {
    RowsRaw<XK> x[MT];
    // float rows are asked for before the weight, and rounded while it is on its way
    if constexpr (XK != kRows8) {
#pragma unroll
      for (int j = 0; j < MT; ++j) load_rows<XK>(p, m0 + 16 * j, kb, lane, x[j]);
    }
    i32x8_ a[NT];
    const int sa = *reinterpret_cast<const int*>(st + (int64_t)kb * p.NP * 4);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint8_t* q = wt + ((int64_t)t * p.KB + kb) * 2048;
      a[t] = join8(*reinterpret_cast<const i32x4_*>(q), *reinterpret_cast<const i32x4_*>(q + 1024));
    }
    if constexpr (XK == kRows8) {
#pragma unroll
      for (int j = 0; j < MT; ++j) load_rows<XK>(p, m0 + 16 * j, kb, lane, x[j]);
    }
    i32x8_ b[MT];
    int sb[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) rows_operand<XK>(x[j], p.K - kb * kStep8, lane, b[j], sb[j]);
    if constexpr (!SHORT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // a plane's halves, each 8 k of a lane
        const int sw = plane_scale(sa, lane, i >> 1);
        bf16x8 w[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t] = widen8(a[t], i, sw >> (8 * t));
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const bf16x8 v = widen8(b[j], i, plane_scale(sb[j], lane, i >> 1));
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[t], v, acc[j][t], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        mma8<0, 0>(acc[j][0], a[0], sa, b[j], sb[j]);
        mma8<1, 0>(acc[j][1], a[1], sa, b[j], sb[j]);
        mma8<2, 0>(acc[j][2], a[2], sa, b[j], sb[j]);
        mma8<3, 0>(acc[j][3], a[3], sa, b[j], sb[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) {
#pragma unroll
    for (int t = 0; t < NT; ++t) part[wave][j][t][lane] = acc[j][t];
  }
  __syncthreads();
  // wave j finishes row tile j
  for (int j = wave; j < MT; j += kFewWaves) {
    const int64_t m = m0 + 16 * j + (lane & 15);
    f32x4 v[4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      v[t] = part[0][j][t][lane];
      for (int w = 1; w < kFewWaves; ++w) v[t] += part[w][j][t][lane];
    }
    if (m >= p.M) continue;
    finish_group<GATED>(p, m, tile0 / 4, lane, v);
  }
}

// ---- many rows --------------------------------------------------------------------------
// Tiles of 32 x 32: 32 rows of the weight are two packed tiles, and a step of 64 k one of their planes, of
// which lane l (c = l & 31, h = l >> 5) has row c's k 16 h .. and 32 + 16 h ... Four
// v_mfma_f32_32x32x16_bf16 take 8 k of either half each, with the scales of both blocks of row c; one
// v_mfma_scale_f32_32x32x64_f8f6f4 (short sums) takes all 64, with the scale of block h. Three widenings of
// two values to a product lie under it (8192^3: 763 us, 1.44 PFLOP/s, the library's in bf16 1.27; short sums
// 392). A workgroup of four waves takes 32 TN WN outputs (packed rows) and
// 32 TM WM rows. Each step of 64 k goes to LDS by direct loads as the lanes will read it, in planes of
// 16 bytes a lane, two steps ahead of its products in a ring of three stages; the scales go to
// registers. Two workgroups share a CU, so that one's loads, outputs and gates run under the
// other's products: with one of 256 x 256 outputs there they stood in line (16384 x 1024 x 4480:
// 104 us, of them 31 for the outputs and some 25 until a tile's first products).
constexpr int kBand = 16;
// Outputs past the L2s (8 of 4 MB) go by them: kept there they push out the operands, and are gone when
// they are read again. (us with short sums, 16384 x 1024 x 4480 over rotating buffers 106, so 75; 8192 rows 50, 41;
// a model's forward of 16384 tokens, d_model 2048, 3500, 3430; d_model 1024, which reads 147 MB back at once,
// 1715, 1724. With float32 sums, whose products take as long as the outputs, either way is the same within
// 2%: 8192 rows 73, 71; 32768 x 2048 x 1024 with a residual 123, 123.)
constexpr int64_t kPastCache = 32 << 20;
__device__ __forceinline__ void store_once(const M8Params& p, bf16* to, bf16x8 o) {
  if (p.vec & 4) {
    asm volatile("" ::: "memory");   // else the two stores become a plain one
    __builtin_nontemporal_store(o, reinterpret_cast<bf16x8*>(to));
    asm volatile("" ::: "memory");
  } else {
    *reinterpret_cast<bf16x8*>(to) = o;
  }
}
typedef float f32x16 __attribute__((ext_vector_type(16)));

// A wave's accumulators: group q's tile T and row tile j; element 4 u + e of lane (c, h) is row
// 32 j + c and output 64 q + 32 T + 16 (u & 1) + 8 h + 4 (u >> 1) + e (gated: 32 q + ... of value or gate).
template <int TN, int TM, bool GATED>
__device__ __forceinline__ void finish_tile(const M8Params& p, const f32x16 (&acc)[TN][TM], int grp0,
                                            int64_t row0, bool plain, int lane, float* sh) {
  const int c = lane & 31, h = lane >> 5;
  if constexpr (GATED) {
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int64_t m = row0 + 32 * j + c;
#pragma unroll
      for (int q = 0; q < TN / 2; ++q) {
        const int grp = grp0 + q;
        if (m < p.M && grp < p.NP / 64) {   // both lanes of a row
          float v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {   // i: 8 outputs from 8 h, then 8 from 16 + 8 h
            const int e = 8 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3);
            float a = acc[2 * q][j][e], b = acc[2 * q + 1][j][e];
            if (p.bias) {
              const int n = min(32 * grp + 16 * (i >> 3) + 8 * h + (i & 7), p.N - 1);
              a += p.bias[n];
              b += p.bias[p.N + n];
            }
            v[i] = a * silu8(b);
          }
          if (32 * grp + 32 > p.N) {   // zeros behind the width
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (32 * grp + 16 * (i >> 3) + 8 * h + (i & 7) >= p.N) v[i] = 0.f;
          }
          uint32_t u = max_bits(v), o = (uint32_t)__shfl_xor((int)u, 32, 64);
          u = u > o ? u : o;
          if (u >= kInfBits) {
            u = max_bits_finite(v);
            o = (uint32_t)__shfl_xor((int)u, 32, 64);
            u = u > o ? u : o;
          }
          const int byte = scale_byte(u);
          const float down = scale_down(byte);
          uint8_t* out = p.yv + value_at(m, 32 * grp + 8 * h, p.NP / 256);
          *reinterpret_cast<i32x2_*>(out) = i32x2_{pack4(v[0], v[1], v[2], v[3], down), pack4(v[4], v[5], v[6], v[7], down)};
          *reinterpret_cast<i32x2_*>(out + 256) =   // 16 k on
              i32x2_{pack4(v[8], v[9], v[10], v[11], down), pack4(v[12], v[13], v[14], v[15], down)};
          if (h == 0) p.ys[(int64_t)grp * p.mp + scale_at(m)] = (uint8_t)byte;
        }
      }
    }
  } else if (plain) {
    // No activation: turned in LDS, and out as whole 16-byte pieces of rows, 64 TN bytes of a row behind
    // each other. From the accumulators alone a store's lanes hold 32 bytes of each of 32 rows
    // (16384 x 1024 x 4480: 103 us, so 87). Without a residual LDS holds the outputs' own bf16; with one
    // float32, as the sum is rounded once, and the residual's rows are read a turn ahead (16384 x 2048 x 1024:
    // 35.9 us, so 35.0; all of a tile's at once 37.4).
    if (p.residual) {
      constexpr int W = 32 * TN, LD = W + 4, PR = W / 8, RI = 64 / PR;
      const int n0 = 64 * grp0, piece = lane % PR, n = n0 + 8 * piece;
      float bias[8] = {};
      if (p.bias && n < p.N) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p.bias + n), d = *reinterpret_cast<const f32x4*>(p.bias + n + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { bias[i] = a[i]; bias[4 + i] = d[i]; }
      }
      bf16x8 res_[2][32 / RI];
      auto fetch = [&](int j, bf16x8 (&to)[32 / RI]) {
#pragma unroll
        for (int i = 0; i < 32 / RI; ++i) {
          const int64_t m = row0 + 32 * j + lane / PR + RI * i;
          to[i] = m < p.M && n < p.N ? *reinterpret_cast<const bf16x8*>(p.residual + m * p.ldr + n) : bf16x8{};
        }
      };
      fetch(0, res_[0]);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const int64_t mj = row0 + 32 * j + lane / PR;
        auto& res = res_[j & 1];
        if (j + 1 < TM) fetch(j + 1, res_[(j + 1) & 1]);
#pragma unroll
        for (int t = 0; t < TN; ++t) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            *reinterpret_cast<f32x4*>(sh + c * LD + 32 * t + 16 * (u & 1) + 8 * h + 4 * (u >> 1)) =
                f32x4{acc[t][j][4 * u], acc[t][j][4 * u + 1], acc[t][j][4 * u + 2], acc[t][j][4 * u + 3]};
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < 32 / RI; ++i) {
          const int64_t m = mj + RI * i;
          const float* from = sh + (i * RI + lane / PR) * LD + 8 * piece;
          const f32x4 a = *reinterpret_cast<const f32x4*>(from), d = *reinterpret_cast<const f32x4*>(from + 4);
          bf16x8 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[e] = (bf16)(a[e] + bias[e] + (float)res[i][e]);
            o[4 + e] = (bf16)(d[e] + bias[4 + e] + (float)res[i][4 + e]);
          }
          if (m < p.M && n < p.N) store_once(p, p.y + m * p.ldy + n, o);
        }
        wave_sync();
      }
      return;
    }
    constexpr int W = 32 * TN, LD = W + 8, PR = W / 8, RI = 64 / PR;   // pieces a row, rows at once
    bf16* sb = reinterpret_cast<bf16*>(sh);
    const int n0 = 64 * grp0, piece = lane % PR, n = n0 + 8 * piece;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
#pragma unroll
      for (int t = 0; t < TN; ++t) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = 32 * t + 16 * k + 8 * h;
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = acc[t][j][8 * (i >> 2) + 4 * k + (i & 3)];
          if (p.bias && n0 + at < p.N) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p.bias + n0 + at);
            const f32x4 d = *reinterpret_cast<const f32x4*>(p.bias + n0 + at + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] += a[i]; v[4 + i] += d[i]; }
          }
          bf16x8 o;
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = (bf16)v[i];
          *reinterpret_cast<bf16x8*>(sb + c * LD + at) = o;
        }
      }
      wave_sync();
      const int64_t mj = row0 + 32 * j + lane / PR;
      bf16* yr = p.y + mj * p.ldy + n;
#pragma unroll
      for (int i = 0; i < 32 / RI; ++i) {
        const bf16x8 o = *reinterpret_cast<const bf16x8*>(sb + (i * RI + lane / PR) * LD + 8 * piece);
        if (mj + RI * i < p.M && n < p.N) store_once(p, yr + (int64_t)(RI * i) * p.ldy, o);
      }
      wave_sync();
    }
  } else {
    // 32 rows at a time through the wave's share of LDS, so that odd widths and the activations are one
    // loop each, and not unrolled over every accumulator
    constexpr int W = 32 * TN, LD = W + 4;
    const int n0 = 64 * grp0;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
#pragma unroll
      for (int t = 0; t < TN; ++t) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          *reinterpret_cast<f32x4*>(sh + c * LD + 32 * t + 16 * (u & 1) + 8 * h + 4 * (u >> 1)) =
              f32x4{acc[t][j][4 * u], acc[t][j][4 * u + 1], acc[t][j][4 * u + 2], acc[t][j][4 * u + 3]};
      }
      wave_sync();
      const int64_t mj = row0 + 32 * j;
      if (p.vec & 1) {
#pragma unroll 1
        for (int e = lane; e < 32 * (W / 8); e += 64) {
          const int row = e / (W / 8), n = 8 * (e % (W / 8));
          if (mj + row < p.M) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(sh + row * LD + n);
            const f32x4 d = *reinterpret_cast<const f32x4*>(sh + row * LD + n + 4);
            float v[8] = {a[0], a[1], a[2], a[3], d[0], d[1], d[2], d[3]};
            finish8(p, mj + row, n0 + n, v);
          }
        }
      } else {
#pragma unroll 1
        for (int e = lane; e < 32 * W; e += 64) {
          const int row = e / W, n = n0 + e % W;
          const int64_t m = mj + row;
          if (m < p.M && n < p.N) {
            float v = sh[row * LD + e % W];
            if (p.bias) v += p.bias[n];
            v = act8(v, p.act);
            if (p.residual) v += (float)p.residual[m * p.ldr + n];
            p.y[m * p.ldy + n] = (bf16)v;
          }
        }
      }
      wave_sync();
    }
  }
}

template <int WN, int WM, int TN, int TM, bool GATED, bool SHORT>
__global__ void __launch_bounds__(64 * WN * WM, 2) matmul8_kernel(const M8Params p) {
  constexpr int NW = WN * WM, NTL = 2 * TN * WN, MTL = 2 * TM * WM;   // 16-row tiles
  constexpr int LN = NTL / NW, LM = MTL / NW;    // tiles whose plane a wave loads
  constexpr int NS = SHORT ? 1 : 2;              // scales of a lane's row: its half's block, or both blocks
  constexpr int kOps = LN + LM + NS * (TN / 2 + 1);   // vector memory operations of a step's loads
  static_assert(NTL % NW == 0 && MTL % NW == 0 && TN % 2 == 0 && (TM == 1 || TM == 2 || TM == 4), "tiles");
  constexpr int kStageBytes = (NTL + MTL) * 1024, kShare = 32 * (32 * TN + 4) * 4;
  constexpr int kLds = 3 * kStageBytes > NW * kShare || GATED ? 3 * kStageBytes : NW * kShare;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // One XCD's workgroups take consecutive tiles, kBand row tiles high and walked along the outputs:
  // the 64 at work at a time read some 16 strips of rows and 4 of the weight through their L2, where
  // one row tile's would read as many strips of the weight as there are workgroups (8192^3, 256 x 256
  // outputs to a workgroup: 540 us, with bands 447).
  const int nb = p.tiles_m * p.tiles_n, per = (nb + 7) >> 3, bid = blockIdx.x;
  const int lin = (bid & 7) * per + (bid >> 3);
  if (lin >= nb) return;
  const int band = lin / (kBand * p.tiles_n), high = min(kBand, p.tiles_m - band * kBand);
  const int at = lin - band * kBand * p.tiles_n;
  const int ntiles = p.NP / 16, tile0 = at / high * NTL;
  const int64_t m0 = (int64_t)(band * kBand + at % high) * (16 * MTL);
  const uint32_t wstep = (uint32_t)p.KB * 2048;
  const uint8_t* wbase = p.w + (int64_t)tile0 * wstep;
  const uint8_t* xbase = static_cast<const uint8_t*>(p.x) + (m0 >> 4) * wstep;
  const int S = 2 * p.KB;
  const int wn = wave % WN, wm = wave / WN, c = lane & 31, h = lane >> 5;
  const int rtiles = (int)min((p.M - m0 + 15) >> 4, (int64_t)MTL);
  // a tile behind the last reads the last one instead, and is not stored
  uint32_t ow[LN], ox[LM];
#pragma unroll
  for (int i = 0; i < LN; ++i) ow[i] = (uint32_t)min(wave * LN + i, ntiles - 1 - tile0) * wstep + 16 * lane;
#pragma unroll
  for (int i = 0; i < LM; ++i) ox[i] = (uint32_t)min(wave * LM + i, rtiles - 1) * wstep + 16 * lane;
  // Behind the last step the loads go through empty descriptors, at offsets that lie in the operands
  // whatever the range check makes of a uniform one, and touch no memory.
  auto load = [&](int stage, int s) {
    s = __builtin_amdgcn_readfirstlane(s);
    const uint32_t bytes = s < S ? 0xfffffff0u : 0u, from = (uint32_t)step_within(s, S) * 1024;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(wbase, bytes), rx = make_rsrc(xbase, bytes);
    uint8_t* to = lds + stage * kStageBytes;
#pragma unroll
    for (int i = 0; i < LN; ++i) buf_load_lds16(rw, to + (wave * LN + i) * 1024, ow[i], from);
#pragma unroll
    for (int i = 0; i < LM; ++i) buf_load_lds16(rx, to + (NTL + wave * LM + i) * 1024, ox[i], from);
  };
  // group q's dword holds its four 16-row tiles' scales of a row; bit 4 of the lane picks the tile of a pair
  const int grp0 = tile0 / 4 + TN / 2 * wn;
  uint32_t osw[TN / 2];
#pragma unroll
  for (int q = 0; q < TN / 2; ++q) osw[q] = weight_scale_at(grp0 + q, p.NP / 64, (SHORT ? 16 * h : 0) + (lane & 15));
  const int64_t mw = m0 + 32 * TM * wm;   // the wave's rows
  const uint32_t osx = (uint32_t)((SHORT ? (int64_t)h * p.mp : 0) + (mw & ~(int64_t)127) + 4 * c);
  auto scales = [&](int s, int (&sw)[TN / 2][NS], int (&sx)[NS]) {
    s = __builtin_amdgcn_readfirstlane(s);
    const int at = step_within(s, S);
    const __amdgpu_buffer_rsrc_t rws = make_rsrc(p.ws, s < S ? (uint32_t)((int64_t)p.KB * p.NP * 4) : 0u);
    const __amdgpu_buffer_rsrc_t rxs = make_rsrc(p.xs, s < S ? (uint32_t)((int64_t)p.KB * p.mp * 4) : 0u);
#pragma unroll
    for (int e = 0; e < NS; ++e) {
#pragma unroll
      for (int q = 0; q < TN / 2; ++q)
        sw[q][e] = __builtin_amdgcn_raw_buffer_load_b32(rws, osw[q], weight_scale_step(at, p.NP) + 64 * e, 0);
      sx[e] = __builtin_amdgcn_raw_buffer_load_b32(rxs, osx, (uint32_t)((int64_t)(2 * at + e) * p.mp), 0);
    }
  };
  f32x16 acc[TN][TM];
#pragma unroll
  for (int t = 0; t < TN; ++t) {
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[t][j] = f32x16{};
  }
  int sw[3][TN / 2][NS], sx[3][NS];
  // half h's k of tile pair T: lane group 2 half + h of plane, rows c of both tiles
  const int lread = (c >> 4) * 1024 + h * 256 + (c & 15) * 16;
  auto step = [&](auto rc, auto behind, int s) {
    constexpr int R = decltype(rc)::value;
    // This step's loads are done when only the next one's are under way; every wave has read the stage
    // that the loads of the step after that fill. The count holds where each step of the loop before it
    // asked for its kOps, which the loop's carried registers keep alive; the last steps, behind the loop,
    // ask for nothing more and wait for all.
    constexpr bool kLast = decltype(behind)::value;
    if constexpr (kLast) vm_wait_all();
    else vm_wait_keep<kOps>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const uint8_t* at = lds + R * kStageBytes + lread;
    auto frag = [&](int tile) {
      return join8(*reinterpret_cast<const i32x4_*>(at + tile * 2048),
                   *reinterpret_cast<const i32x4_*>(at + tile * 2048 + 512));
    };
    i32x8_ a[TN], b[TM];
#pragma unroll
    for (int t = 0; t < TN; ++t) a[t] = frag(wn * TN + t);
#pragma unroll
    for (int j = 0; j < TM; ++j) b[j] = frag(NTL / 2 + wm * TM + j);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!kLast) load((R + 2) % 3, s + 2);
    const int by = 8 * (c >> 4), bx = 8 * ((int)(mw >> 5) & 3);
    if constexpr (SHORT) {
      const int sr = (int)((uint32_t)sx[R][0] >> bx);
#pragma unroll
      for (int q = 0; q < TN / 2; ++q) {
        const int s4 = (int)((uint32_t)sw[R][q][0] >> by);
        static_for<TM>([&](auto jc) {
          constexpr int j = decltype(jc)::value;
          acc[2 * q][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[2 * q], b[j], acc[2 * q][j], 0, 0, 0, s4, j, sr);
          acc[2 * q + 1][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[2 * q + 1], b[j], acc[2 * q + 1][j], 0, 0, 2, s4, j, sr);
        });
      }
      // the loads between the products, and not before the first of them
#pragma unroll
      for (int i = 0; i < TN * TM; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x010, (LN + LM + TN * TM - 1) / (TN * TM), 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // 8 k of either half, of block i >> 1
        bf16x8 wa[TN];
#pragma unroll
        for (int t = 0; t < TN; ++t) wa[t] = widen8(a[t], i, sw[R][t / 2][i >> 1] >> (by + 16 * (t & 1)));
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const bf16x8 xb = widen8(b[j], i, sx[R][i >> 1] >> (bx + 8 * j));
#pragma unroll
          for (int t = 0; t < TN; ++t) acc[t][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wa[t], xb, acc[t][j], 0, 0, 0);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!kLast) scales(s + 3, sw[R], sx[R]);
    asm volatile("" ::: "memory");
  };
  const std::integral_constant<int, 0> r0;
  const std::integral_constant<int, 1> r1;
  const std::integral_constant<int, 2> r2;
  // in this order: a step counts the operations behind its own loads
  scales(0, sw[0], sx[0]);
  load(0, 0);
  __builtin_amdgcn_sched_barrier(0);
  scales(1, sw[1], sx[1]);
  load(1, 1);
  scales(2, sw[2], sx[2]);
  __builtin_amdgcn_sched_barrier(0);
  int s = 0;
  for (; s + 3 <= S; s += 3) {   // no way out in the middle: the compiler would wait for scales just asked for
    step(r0, std::false_type{}, s);
    step(r1, std::false_type{}, s + 1);
    step(r2, std::false_type{}, s + 2);
  }
  if (s < S) step(r0, std::true_type{}, s);
  if (s + 1 < S) step(r1, std::true_type{}, s + 1);
  vm_wait_all();   // no load may reach LDS behind the workgroup's end
  const bool plain = (p.vec & 1) && p.act == kActNone && p.N % 8 == 0;
  if (!GATED) __syncthreads();
  finish_tile<TN, TM, GATED>(p, acc, (tile0 + 2 * TN * wn) / 4, m0 + 32 * TM * wm, plain, lane,
                             reinterpret_cast<float*>(lds) + wave * (kShare / 4));
}

template <int MT, int XK, bool GATED, bool SHORT>
static void launch_few(const M8Params& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.NP / 64), (unsigned)((p.M + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((matmul8_few_kernel<MT, XK, GATED, SHORT>), grid, dim3(64 * kFewWaves), 0, s, p);
}

template <int WN, int WM, int TN, int TM, bool GATED, bool SHORT>
static void launch_many(M8Params p, hipStream_t s) {
  p.tiles_n = (p.NP + 32 * TN * WN - 1) / (32 * TN * WN);
  p.tiles_m = (int)((p.M + 32 * TM * WM - 1) / (32 * TM * WM));
  const int64_t nb = (int64_t)p.tiles_m * p.tiles_n;
  const unsigned grid = (unsigned)(((nb + 7) >> 3) * 8);
  hipLaunchKernelGGL((matmul8_kernel<WN, WM, TN, TM, GATED, SHORT>), dim3(grid), dim3(64 * WN * WM), 0, s, p);
}

template <bool GATED, bool SHORT>
static void dispatch8(const M8Params& p, int x_dtype, hipStream_t s) {
  if (x_dtype == M3S_DTYPE_BF16) return launch_few<1, kRowsBf16, GATED, SHORT>(p, s);
  if (x_dtype == M3S_DTYPE_F32) return launch_few<1, kRowsF32, GATED, SHORT>(p, s);
  switch (form8(p.M, p.NP)) {
    case kFew16: return launch_few<1, kRows8, GATED, SHORT>(p, s);
    case kFew32: return launch_few<2, kRows8, GATED, SHORT>(p, s);
    case kTiles64: return launch_many<2, 2, 2, 1, GATED, SHORT>(p, s);
    case kTiles64Wide: return launch_many<4, 1, 2, 2, GATED, SHORT>(p, s);
    case kTiles128: return launch_many<4, 1, 2, 4, GATED, SHORT>(p, s);
  }
}

}  // namespace m3s

using namespace m3s;

static int packed_outputs(int32_t n, bool gated) {
  return (int)(gated ? 2 * padded8(n) : ((int64_t)n + 63) / 64 * 64);
}

extern "C" int32_t m3s_matmul8_takes_floats(int64_t rows, int32_t k, int32_t n, int32_t gated, int32_t x_dtype) {
  if (rows < 0 || k < 1 || k > M3S_ROWS8_WIDTH_MAX || n < 1 || n > M3S_ROWS8_WIDTH_MAX) return 0;
  if (x_dtype != M3S_DTYPE_BF16 && x_dtype != M3S_DTYPE_F32) return 0;
  return rounds_in_launch(rows, packed_outputs(n, gated != 0), k, x_dtype == M3S_DTYPE_F32 ? 4 : 2);
}

extern "C" int32_t m3s_matmul8(const m3s_matmul8_args* a, void* stream) {
  clear_error();
  M3S_REQUIRE(a != nullptr, "m3s_matmul8: args is NULL");
  M3S_REQUIRE(a->struct_size == (int32_t)sizeof(m3s_matmul8_args),
              "m3s_matmul8: struct_size %d != %d (ABI mismatch)", a->struct_size,
              (int)sizeof(m3s_matmul8_args));
  M3S_REQUIRE(a->x_dtype == M3S_DTYPE_BF16 || a->x_dtype == M3S_DTYPE_F32 || a->x_dtype == M3S_DTYPE_ROWS8,
              "m3s_matmul8: bad x_dtype %d", a->x_dtype);
  M3S_REQUIRE(a->activation >= M3S_ACT_NONE && a->activation <= M3S_ACT_RELU, "m3s_matmul8: bad activation %d",
              a->activation);
  M3S_REQUIRE(a->rows >= 0 && a->rows <= M3S_ROWS8_MAX, "m3s_matmul8: rows %lld out of range", (long long)a->rows);
  M3S_REQUIRE(a->k > 0 && a->k <= M3S_ROWS8_WIDTH_MAX && a->n > 0 && a->n <= M3S_ROWS8_WIDTH_MAX,
              "m3s_matmul8: k %d or n %d out of range", a->k, a->n);
  const bool floats = a->x_dtype != M3S_DTYPE_ROWS8;
  M3S_REQUIRE(!floats || a->rows <= M3S_MATMUL8_FLOAT_ROWS, "m3s_matmul8: %lld rows in floating point, over %d",
              (long long)a->rows, M3S_MATMUL8_FLOAT_ROWS);
  if (a->rows == 0) return 0;
  M3S_REQUIRE(a->x && a->w && a->w_scales && (floats || a->x_scales), "m3s_matmul8: NULL pointer");
  M3S_REQUIRE(a->gated ? (a->y_values && a->y_scales && !a->y && !a->residual && a->activation == M3S_ACT_NONE)
                       : (a->y && !a->y_values && !a->y_scales),
              "m3s_matmul8: a gated product takes y_values and y_scales alone, another y");
  M3S_REQUIRE(aligned16(a->w) && (floats || aligned16(a->x)) && (!a->gated || aligned16(a->y_values)),
              "m3s_matmul8: 8-bit values must be 16-byte aligned");
  M3S_REQUIRE((uintptr_t)a->w_scales % 4 == 0 && (floats || (uintptr_t)a->x_scales % 4 == 0),
              "m3s_matmul8: scales must be 4-byte aligned");
  M3S_REQUIRE(!floats || a->ldx >= a->k, "m3s_matmul8: ldx is too short");
  M3S_REQUIRE(!a->residual || a->ldres >= a->n, "m3s_matmul8: ldres is too short");
  M3S_REQUIRE(a->gated || a->ldy >= a->n, "m3s_matmul8: ldy is too short");
  M8Params p{};
  p.x = a->x; p.xs = static_cast<const uint8_t*>(a->x_scales);
  p.w = static_cast<const uint8_t*>(a->w); p.ws = static_cast<const uint8_t*>(a->w_scales);
  p.bias = a->bias; p.residual = static_cast<const bf16*>(a->residual); p.y = static_cast<bf16*>(a->y);
  p.yv = static_cast<uint8_t*>(a->y_values); p.ys = static_cast<uint8_t*>(a->y_scales);
  p.M = a->rows; p.mp = padded_rows(a->rows); p.ldx = a->ldx; p.ldr = a->ldres; p.ldy = a->ldy;
  p.K = a->k; p.KB = (int)(padded8(a->k) / kStep8); p.N = a->n; p.act = a->activation;
  p.NP = packed_outputs(a->n, a->gated != 0);
  // scales are read through 32-bit offsets, and a launch holds at most 2^31 workgroups' tiles
  M3S_REQUIRE((int64_t)p.KB * p.mp * 4 < (1ll << 31) && (int64_t)p.KB * p.NP * 4 < (1ll << 31),
              "m3s_matmul8: an operand's scales span 2 GiB or more");
  const bool whole = p.ldy % 8 == 0 && aligned16(p.y) && (!p.bias || aligned16(p.bias)) &&
                     (!p.residual || (aligned16(p.residual) && p.ldr % 8 == 0));
  const int xs = a->x_dtype == M3S_DTYPE_F32 ? 4 : 2;
  const bool xvec = floats && p.K % 8 == 0 && aligned16(p.x) && p.ldx % (16 / xs) == 0;
  p.vec = (whole ? 1 : 0) | (xvec ? 2 : 0) | (a->rows * (int64_t)a->n * 2 > kPastCache ? 4 : 0);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->gated) a->short_sums ? dispatch8<true, true>(p, a->x_dtype, s) : dispatch8<true, false>(p, a->x_dtype, s);
  else a->short_sums ? dispatch8<false, true>(p, a->x_dtype, s) : dispatch8<false, false>(p, a->x_dtype, s);
  return launch_status("m3s_matmul8");
}
