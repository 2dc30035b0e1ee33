// Products of rows and weights in 8 bits on gfx950 (m3s_eight.h), with bias, activation and residual,
// or the MLP's gate and its rows in 8 bits again, in the epilogue:
//
//   y = act(x w + bias) + residual                    in bf16
//   a = value silu(gate), value | gate = x w + bias   in 8 bits, the next product's rows
//
// They stand for the projections of the LM (layer.py:233, 256; model.py:125-140, 231) on weights in
// 8 bits.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 128 k at twice bf16's rate and applies a scale for
// every 32 of them on the way. Its A operand is the weight and its B operand the rows, so a lane's
// four accumulators are four neighbouring outputs of one row. Lane l (r = l & 15, g = l >> 4) gives
// row r's k 16 g .. 16 g + 15 and 64 + 16 g .. of the 128, and the scale of its k 32 g .. 32 g + 31.
// Its sums are short of float32's: of each 8 neighbouring products it cuts what is below 2^-13 of the
// largest one's power of two, and adds the rest to the float32 accumulator (found with pairs of
// products; groups of 8 do not touch each other). A product of N(0, 1) rows is 1.3e-5 off for any
// K from 1024 to 16384, a 150th of a bf16 rounding and a thousandth of e4m3's: that is why products
// leave in bf16 or 8 bits. The float32 route, e4m3 widened to bf16 and multiplied at half the rate,
// would sum in full and round its operands no better.
//
// Weights are packed once (eightbit.pack8): 16-row tiles of 2048 bytes a step, as two planes of 16
// bytes a lane, so that a wave's load is 1 KB in one piece, straight to registers or LDS. Four
// tiles are a group of 64 outputs: tile t, row 4 g + i is output 64 grp + 32 (t >> 1) + 8 g +
// 4 (t & 1) + i, which leaves a lane 8 neighbouring outputs (16 bytes of bf16) in two tiles, and four
// lanes the 32 of a block. With a gate, tiles 0 and 1 hold value's outputs 32 grp + 8 g + 4 t + i and
// tiles 2 and 3 gate's, so a lane has both.
#include <type_traits>

#include "m3s_eight.h"
#include "m3s_internal.h"

namespace m3s {

enum Act8 { kActNone = M3S_ACT_NONE, kActSilu = M3S_ACT_SILU, kActGelu = M3S_ACT_GELU, kActRelu = M3S_ACT_RELU };

struct M8Params {
  const void* x;           // (M, kp) e4m3, or (M, K) bf16 / float32 for few rows
  const uint8_t* xs;       // (4 KB, mp)
  const uint8_t* w;        // [n tile][step][2][lane][16]
  const uint8_t* ws;       // [step][group of four tiles][lane][4]
  const float* bias;
  const bf16* residual;
  bf16* y;
  uint8_t* yv;             // gated: (M, op) values and (op / 32, mp) scales
  uint8_t* ys;
  int64_t M, mp, ldx, ldr, ldy;
  int K, KB, N, NP, act, vec;   // N: outputs (half the weight's columns with a gate); NP: packed rows
  int tiles_m, tiles_n;
};

__device__ __forceinline__ float silu8(float v) { return v / (1.f + __expf(-v)); }
__device__ __forceinline__ float act8(float v, int act) {
  if (act == kActSilu) return silu8(v);
  if (act == kActGelu) return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
  if (act == kActRelu) return v > 0.f ? v : (v == v ? 0.f : v);
  return v;
}

__device__ __forceinline__ uint32_t max_lanes16(uint32_t u) {   // over the four lanes of a row
  uint32_t o = (uint32_t)__shfl_xor((int)u, 16, 64);
  u = u > o ? u : o;
  o = (uint32_t)__shfl_xor((int)u, 32, 64);
  return u > o ? u : o;
}

// 8 neighbouring outputs n .. n + 7 of row m. PLAIN: all there, 16 bytes at once, no activation.
template <bool PLAIN>
__device__ __forceinline__ void finish8(const M8Params& p, int64_t m, int n, float (&v)[8]) {
  if (!PLAIN && n >= p.N) return;
  const bool whole = PLAIN || ((p.vec & 1) && n + 8 <= p.N);   // pointers and strides allow 16 bytes
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
  if (!PLAIN && p.act != kActNone) {
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
template <bool GATED, bool PLAIN>
__device__ __forceinline__ void finish_group(const M8Params& p, int64_t m, int grp, int lane,
                                             const f32x4 (&acc)[4]) {
  const int g = lane >> 4;
  if constexpr (!GATED) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[i] = acc[2 * h][i]; v[4 + i] = acc[2 * h + 1][i]; }
      finish8<PLAIN>(p, m, 64 * grp + 32 * h + 8 * g, v);
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
    const int64_t op = (int64_t)(p.NP / 256) * kStep8;
    *reinterpret_cast<i32x2_*>(p.yv + m * op + j) =
        i32x2_{pack4(v[0], v[1], v[2], v[3], down), pack4(v[4], v[5], v[6], v[7], down)};
    if (g == 0) p.ys[(int64_t)grp * p.mp + m] = (uint8_t)byte;
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
// a row of products: tile t of the weight (its byte of sa) with the TM row tiles
template <int T, int TM>
__device__ __forceinline__ void mma8_rows(f32x4 (&acc)[TM], i32x8_ a, int sa, const i32x8_ (&b)[TM],
                                          const int (&sb)[(TM + 3) / 4]) {
#pragma unroll
  for (int q = 0; q < (TM + 3) / 4; ++q) {
    mma8<T, 0>(acc[4 * q], a, sa, b[4 * q], sb[q]);
    if constexpr (TM > 1) mma8<T, 1>(acc[4 * q + 1], a, sa, b[4 * q + 1], sb[q]);
    if constexpr (TM > 2) mma8<T, 2>(acc[4 * q + 2], a, sa, b[4 * q + 2], sb[q]);
    if constexpr (TM > 3) mma8<T, 3>(acc[4 * q + 3], a, sa, b[4 * q + 3], sb[q]);
  }
}

// ---- few rows ---------------------------------------------------------------------------
// The weight is the traffic. A workgroup takes a group of 64 outputs and 16 MT rows; its eight waves take the steps of K in turn, each loading its tiles straight to
// registers, and their sums meet in LDS in wave order (deterministic). Float rows are rounded to 8
// bits on the way in: a block is two lanes' half rows.
constexpr int kFewWaves = 8;
enum Rows8Kind { kRows8 = 0, kRowsBf16 = 1, kRowsF32 = 2 };

// lane's operand and scale of rows m .. m + 15, step kb
template <int XK>
__device__ __forceinline__ void rows_operand(const M8Params& p, int64_t m0, int kb, int lane, i32x8_& b, int& sb) {
  const int r = lane & 15, g = lane >> 4;
  const int64_t m = m0 + r;
  if constexpr (XK == kRows8) {
    const int64_t mc = m < p.M ? m : p.M - 1;
    const uint8_t* xr = static_cast<const uint8_t*>(p.x) + mc * ((int64_t)p.KB * kStep8) + kb * kStep8 + 16 * g;
    b = join8(*reinterpret_cast<const i32x4_*>(xr), *reinterpret_cast<const i32x4_*>(xr + 64));
    sb = p.xs[((int64_t)kb * 4 + g) * p.mp + mc];
  } else {
    using TX = std::conditional_t<XK == kRowsBf16, bf16, float>;
    int q[8], byte[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = kb * kStep8 + 64 * h + 16 * g;
      float v[16];
      if (m < p.M) {
        const TX* xr = static_cast<const TX*>(p.x) + m * p.ldx + c;
        if (p.vec & 2) {   // whole pieces of 16 bytes; K % 8 == 0
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            if (c + e < p.K) {
              if constexpr (XK == kRowsBf16) {
                const bf16x8 t = *reinterpret_cast<const bf16x8*>(xr + e);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[e + i] = (float)t[i];
              } else {
                const f32x4 t = *reinterpret_cast<const f32x4*>(xr + e), s = *reinterpret_cast<const f32x4*>(xr + e + 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) { v[e + i] = t[i]; v[e + 4 + i] = s[i]; }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) v[e + i] = 0.f;
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = c + i < p.K ? (float)xr[i] : 0.f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.f;
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

template <int MT, int XK, bool GATED>
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
    i32x8_ a[NT];
    const int sa = *reinterpret_cast<const int*>(st + (int64_t)kb * p.NP * 4);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint8_t* q = wt + ((int64_t)t * p.KB + kb) * 2048;
      a[t] = join8(*reinterpret_cast<const i32x4_*>(q), *reinterpret_cast<const i32x4_*>(q + 1024));
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      i32x8_ b;
      int sb;
      rows_operand<XK>(p, m0 + 16 * j, kb, lane, b, sb);
      mma8<0, 0>(acc[j][0], a[0], sa, b, sb);
      mma8<1, 0>(acc[j][1], a[1], sa, b, sb);
      mma8<2, 0>(acc[j][2], a[2], sa, b, sb);
      mma8<3, 0>(acc[j][3], a[3], sa, b, sb);
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
    finish_group<GATED, false>(p, m, tile0 / 4, lane, v);
  }
}

// ---- many rows --------------------------------------------------------------------------
// A workgroup of WN x WM waves takes 16 TN WN outputs (packed rows) and 16 TM WM rows, a wave TN x TM
// tiles of them in accumulators. Each step's operands go to LDS by direct loads, as the lanes will
// read them: a plane of 16 bytes a lane, so neither the loads nor the reads meet a bank twice. Two
// stages: the loads of the next step, and its scales, are in flight under this one's products. Row
// tile j of four holds rows 4 r + j, so that a lane's four scales are one dword.
template <int WN, int WM, int TN, int TM, bool GATED>
__global__ void __launch_bounds__(64 * WN * WM) matmul8_kernel(const M8Params p) {
  constexpr int NW = WN * WM, NTL = TN * WN, MTL = TM * WM;
  constexpr int LN = NTL / NW, LM = MTL / NW;    // tiles a wave loads
  static_assert(NTL % NW == 0 && MTL % NW == 0 && TN % 4 == 0 && TM % 4 == 0, "whole tiles to a wave");
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][(NTL + MTL) * 2048];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  // the tiles that one XCD works on at a time share rows: its workgroups walk the outputs first
  const int nb = p.tiles_m * p.tiles_n, per = (nb + 7) >> 3, bid = blockIdx.x;
  const int lin = (bid & 7) * per + (bid >> 3);
  if (lin >= nb) return;
  const int tn = lin % p.tiles_n, tm = lin / p.tiles_n;
  const int ntiles = p.NP / 16, tile0 = tn * NTL;
  const int64_t m0 = (int64_t)tm * (16 * MTL);
  const int64_t kp = (int64_t)p.KB * kStep8;
  const uint32_t wstep = (uint32_t)p.KB * 2048;
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w + (int64_t)tile0 * wstep, 0xfffffff0u);
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(static_cast<const uint8_t*>(p.x) + m0 * kp, 0xfffffff0u);
  const __amdgpu_buffer_rsrc_t rws = make_rsrc(p.ws, (uint32_t)((int64_t)p.KB * p.NP * 4));
  const __amdgpu_buffer_rsrc_t rxs = make_rsrc(p.xs, (uint32_t)((int64_t)p.KB * p.mp * 4));
  // a tile behind the last, and a row behind the last, reads the last one instead; neither is stored
  uint32_t ow[LN], ox[LM];
#pragma unroll
  for (int i = 0; i < LN; ++i) ow[i] = (uint32_t)min(wave * LN + i, ntiles - 1 - tile0) * wstep + 16 * lane;
#pragma unroll
  for (int i = 0; i < LM; ++i) {
    const int t = wave * LM + i;
    const int64_t row = min((int64_t)(64 * (t >> 2) + 4 * r + (t & 3)), p.M - 1 - m0);
    ox[i] = (uint32_t)(row * kp) + 16 * g;
  }
  auto load = [&](int buf, int kb) {
#pragma unroll
    for (int i = 0; i < LN; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        buf_load_lds16(rw, lds[buf] + (wave * LN + i) * 2048 + 1024 * h, ow[i] + 1024 * h, (uint32_t)kb * 2048);
    }
#pragma unroll
    for (int i = 0; i < LM; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        buf_load_lds16(rx, lds[buf] + (NTL + wave * LM + i) * 2048 + 1024 * h, ox[i] + 64 * h, (uint32_t)kb * kStep8);
    }
  };
  const int wn = wave % WN, wm = wave / WN;
  const uint32_t osw = (uint32_t)(16 * (tile0 + wn * TN)) * 4 + 4 * lane;
  const uint32_t osx = (uint32_t)((int64_t)g * p.mp + m0 + 16 * wm * TM + 4 * r);
  auto scales = [&](int kb, int (&sw)[TN / 4], int (&sx)[TM / 4]) {
#pragma unroll
    for (int t = 0; t < TN / 4; ++t)
      sw[t] = __builtin_amdgcn_raw_buffer_load_b32(rws, osw + 256 * t, (uint32_t)kb * (uint32_t)p.NP * 4, 0);
#pragma unroll
    for (int j = 0; j < TM / 4; ++j)
      sx[j] = __builtin_amdgcn_raw_buffer_load_b32(rxs, osx + 64 * j, (uint32_t)((int64_t)kb * p.mp * 4), 0);
  };
  f32x4 acc[TN][TM];
#pragma unroll
  for (int t = 0; t < TN; ++t) {
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int sw[TN / 4], sx[TM / 4], sw1[TN / 4], sx1[TM / 4];
  load(0, 0);
  scales(0, sw1, sx1);
  for (int kb = 0; kb < p.KB; ++kb) {
    vm_wait_all();
    __syncthreads();   // this step's stage is whole, and every wave has read the other one
#pragma unroll
    for (int t = 0; t < TN / 4; ++t) sw[t] = sw1[t];
#pragma unroll
    for (int j = 0; j < TM / 4; ++j) sx[j] = sx1[j];
    if (kb + 1 < p.KB) {
      load((kb + 1) & 1, kb + 1);
      scales(kb + 1, sw1, sx1);
    }
    const uint8_t* s = lds[kb & 1] + 16 * lane;
    auto frag = [&](int tile) {
      const uint8_t* q = s + tile * 2048;
      return join8(*reinterpret_cast<const i32x4_*>(q), *reinterpret_cast<const i32x4_*>(q + 1024));
    };
    i32x8_ b[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) b[j] = frag(NTL + wm * TM + j);
#pragma unroll
    for (int q = 0; q < TN / 4; ++q) {
      mma8_rows<0, TM>(acc[4 * q], frag(wn * TN + 4 * q), sw[q], b, sx);
      mma8_rows<1, TM>(acc[4 * q + 1], frag(wn * TN + 4 * q + 1), sw[q], b, sx);
      mma8_rows<2, TM>(acc[4 * q + 2], frag(wn * TN + 4 * q + 2), sw[q], b, sx);
      mma8_rows<3, TM>(acc[4 * q + 3], frag(wn * TN + 4 * q + 3), sw[q], b, sx);
    }
  }
  const int grp0 = (tile0 + wn * TN) / 4;
  const int64_t mw = m0 + 16 * wm * TM + 4 * r;
  // straight from the accumulators where every output of the tile is whole and goes out as it is
  if (GATED || ((p.vec & 1) && p.act == kActNone && 16 * (tile0 + NTL) <= p.N)) {
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int64_t m = mw + 64 * (j >> 2) + (j & 3);
      if (m >= p.M) continue;
#pragma unroll
      for (int q = 0; q < TN / 4; ++q) {
        if (!GATED || grp0 + q < p.NP / 64) {
          const f32x4 v[4] = {acc[4 * q][j], acc[4 * q + 1][j], acc[4 * q + 2][j], acc[4 * q + 3][j]};
          finish_group<GATED, true>(p, m, grp0 + q, lane, v);
        }
      }
    }
    return;
  }
  // else 16 rows at a time through the wave's share of LDS, so that odd widths and the activations are
  // one loop each, and not unrolled over every accumulator
  if constexpr (!GATED) {
    constexpr int LD = 16 * TN + 4;
    static_assert(16 * LD * 4 <= (int)sizeof(lds) / NW, "a wave's 16 rows fit its share");
    __syncthreads();   // the last step's reads
    float* sh = reinterpret_cast<float*>(&lds[0][0]) + wave * (sizeof(lds) / NW / 4);
    const int n0 = 64 * grp0;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
#pragma unroll
      for (int t = 0; t < TN; ++t)
        *reinterpret_cast<f32x4*>(sh + r * LD + 64 * (t >> 2) + 32 * ((t >> 1) & 1) + 8 * g + 4 * (t & 1)) = acc[t][j];
      wave_sync();
      const int64_t mj = m0 + 16 * wm * TM + 64 * (j >> 2) + (j & 3);
      if (p.vec & 1) {
#pragma unroll 1
        for (int e = lane; e < 16 * 2 * TN; e += 64) {
          const int row = e / (2 * TN), c = 8 * (e % (2 * TN));
          if (mj + 4 * row < p.M) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(sh + row * LD + c);
            const f32x4 d = *reinterpret_cast<const f32x4*>(sh + row * LD + c + 4);
            float v[8] = {a[0], a[1], a[2], a[3], d[0], d[1], d[2], d[3]};
            finish8<false>(p, mj + 4 * row, n0 + c, v);
          }
        }
      } else {
#pragma unroll 1
        for (int e = lane; e < 16 * 16 * TN; e += 64) {
          const int row = e / (16 * TN), c = e % (16 * TN);
          const int64_t m = mj + 4 * row;
          const int n = n0 + c;
          if (m < p.M && n < p.N) {
            float v = sh[row * LD + c];
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

template <int MT, int XK, bool GATED>
static void launch_few(const M8Params& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.NP / 64), (unsigned)((p.M + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((matmul8_few_kernel<MT, XK, GATED>), grid, dim3(64 * kFewWaves), 0, s, p);
}

template <int WN, int WM, int TN, int TM, bool GATED>
static void launch_many(M8Params p, hipStream_t s) {
  p.tiles_n = (p.NP / 16 + TN * WN - 1) / (TN * WN);
  p.tiles_m = (int)((p.M + 16 * TM * WM - 1) / (16 * TM * WM));
  const int64_t nb = (int64_t)p.tiles_m * p.tiles_n;
  const unsigned grid = (unsigned)(((nb + 7) >> 3) * 8);
  hipLaunchKernelGGL((matmul8_kernel<WN, WM, TN, TM, GATED>), dim3(grid), dim3(64 * WN * WM), 0, s, p);
}

template <bool GATED>
static void dispatch8(const M8Params& p, int x_dtype, hipStream_t s) {
  if (x_dtype == M3S_DTYPE_BF16) return launch_few<1, kRowsBf16, GATED>(p, s);
  if (x_dtype == M3S_DTYPE_F32) return launch_few<1, kRowsF32, GATED>(p, s);
  if (p.M <= 16) return launch_few<1, kRows8, GATED>(p, s);
  if (p.M <= 256) return launch_few<2, kRows8, GATED>(p, s);
  launch_many<2, 4, 8, 4, GATED>(p, s);
}

}  // namespace m3s

using namespace m3s;

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
  p.M = a->rows; p.mp = padded16(a->rows); p.ldx = a->ldx; p.ldr = a->ldres; p.ldy = a->ldy;
  p.K = a->k; p.KB = (int)(padded8(a->k) / kStep8); p.N = a->n; p.act = a->activation;
  p.NP = (int)(a->gated ? 2 * padded8(a->n) : ((int64_t)a->n + 63) / 64 * 64);
  // scales are read through 32-bit offsets, and a launch holds at most 2^31 workgroups' tiles
  M3S_REQUIRE((int64_t)p.KB * p.mp * 4 < (1ll << 31) && (int64_t)p.KB * p.NP * 4 < (1ll << 31),
              "m3s_matmul8: an operand's scales span 2 GiB or more");
  const bool whole = p.ldy % 8 == 0 && aligned16(p.y) && (!p.bias || aligned16(p.bias)) &&
                     (!p.residual || (aligned16(p.residual) && p.ldr % 8 == 0));
  const int xs = a->x_dtype == M3S_DTYPE_F32 ? 4 : 2;
  const bool xvec = floats && p.K % 8 == 0 && aligned16(p.x) && p.ldx % (16 / xs) == 0;
  p.vec = (whole ? 1 : 0) | (xvec ? 2 : 0);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->gated) dispatch8<true>(p, a->x_dtype, s);
  else dispatch8<false>(p, a->x_dtype, s);
  return launch_status("m3s_matmul8");
}
