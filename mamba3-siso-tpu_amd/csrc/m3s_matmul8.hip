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
  const uint8_t* xs;       // (KB, M, 4)
  const uint8_t* w;        // [n tile][step][2][lane][16]
  const uint8_t* ws;       // (KB, NP, 4)
  const float* bias;
  const bf16* residual;
  bf16* y;
  uint8_t* yv;             // gated: (M, op) values and (op / 128, M, 4) scales
  uint8_t* ys;
  int64_t M, ldx, ldr, ldy;
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

// 8 neighbouring outputs n .. n + 7 of row m
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
      if (p.bias && j + i < p.N) {
        a += p.bias[j + i];
        b += p.bias[p.N + j + i];
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
    if (g == 0) p.ys[((int64_t)(grp >> 2) * p.M + m) * 4 + (grp & 3)] = (uint8_t)byte;
  }
}

__device__ __forceinline__ i32x8_ join8(i32x4_ a, i32x4_ b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ void mma8(f32x4& acc, i32x8_ a, int sa, i32x8_ b, int sb) {
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 0, sa, 0, sb);
}

// ---- few rows ---------------------------------------------------------------------------
// The weight is the traffic. A workgroup takes NT tiles (a group of 64 outputs, or one tile) and
// 16 MT rows; its eight waves take the steps of K in turn, each loading its tiles straight to
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
    sb = p.xs[((int64_t)kb * p.M + mc) * 4 + g];
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

template <int NT, int MT, int XK, bool GATED>
__global__ void __launch_bounds__(64 * kFewWaves) matmul8_few_kernel(const M8Params p) {
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
  const uint8_t* st = p.ws + 64 * tile0 + 4 * (lane & 15) + (lane >> 4);
#pragma unroll 2
  for (int kb = wave; kb < p.KB; kb += kFewWaves) {
    i32x8_ a[NT];
    int sa[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint8_t* q = wt + ((int64_t)t * p.KB + kb) * 2048;
      a[t] = join8(*reinterpret_cast<const i32x4_*>(q), *reinterpret_cast<const i32x4_*>(q + 1024));
      sa[t] = st[(int64_t)kb * p.NP * 4 + 64 * t];
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      i32x8_ b;
      int sb;
      rows_operand<XK>(p, m0 + 16 * j, kb, lane, b, sb);
#pragma unroll
      for (int t = 0; t < NT; ++t) mma8(acc[j][t], a[t], sa[t], b, sb);
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
// A workgroup of WN x WM waves takes 16 TN WN outputs (packed rows) and 16 TM WM rows, a wave TN x TM
// tiles of them in accumulators. Each step's operands go to LDS by direct loads, as the lanes will
// read them: a plane of 16 bytes a lane, so neither the loads nor the reads meet a bank twice. Two
// stages: the loads of the next step are in flight under this one's products.
template <int WN, int WM, int TN, int TM, bool GATED>
__global__ void __launch_bounds__(64 * WN * WM) matmul8_kernel(const M8Params p) {
  constexpr int NW = WN * WM, NTL = TN * WN, MTL = TM * WM;
  constexpr int LN = NTL / NW, LM = MTL / NW;    // tiles a wave loads
  static_assert(NTL % NW == 0 && MTL % NW == 0 && TN % 4 == 0, "whole tiles to a wave");
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
  const __amdgpu_buffer_rsrc_t rxs = make_rsrc(p.xs, (uint32_t)((int64_t)p.KB * p.M * 4));
  // a tile behind the last, and a row behind the last, reads the last one instead; neither is stored
  uint32_t ow[LN], ox[LM];
#pragma unroll
  for (int i = 0; i < LN; ++i) ow[i] = (uint32_t)min(wave * LN + i, ntiles - 1 - tile0) * wstep + 16 * lane;
#pragma unroll
  for (int i = 0; i < LM; ++i) {
    const int64_t row = min((int64_t)(16 * (wave * LM + i) + r), p.M - 1 - m0);
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
  const uint32_t osw = (uint32_t)(16 * (tile0 + wn * TN) + r) * 4 + g;
  const uint32_t osx = (uint32_t)((m0 + 16 * wm * TM + r) * 4 + g);
  int sw[TN], sx[TM];
  auto scales = [&](int kb) {
#pragma unroll
    for (int t = 0; t < TN; ++t)
      sw[t] = __builtin_amdgcn_raw_buffer_load_b8(rws, osw + 64 * t, (uint32_t)kb * p.NP * 4, 0);
#pragma unroll
    for (int j = 0; j < TM; ++j)
      sx[j] = __builtin_amdgcn_raw_buffer_load_b8(rxs, osx + 64 * j, (uint32_t)((int64_t)kb * p.M * 4), 0);
  };
  f32x4 acc[TM][TN];
#pragma unroll
  for (int j = 0; j < TM; ++j) {
#pragma unroll
    for (int t = 0; t < TN; ++t) acc[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  load(0, 0);
  for (int kb = 0; kb < p.KB; ++kb) {
    scales(kb);
    vm_wait_all();
    __syncthreads();   // this step's stage is whole, and every wave has read the other one
    const uint8_t* s = lds[kb & 1] + 16 * lane;
    i32x8_ b[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const uint8_t* q = s + (NTL + wm * TM + j) * 2048;
      b[j] = join8(*reinterpret_cast<const i32x4_*>(q), *reinterpret_cast<const i32x4_*>(q + 1024));
    }
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      const uint8_t* q = s + (wn * TN + t) * 2048;
      const i32x8_ a = join8(*reinterpret_cast<const i32x4_*>(q), *reinterpret_cast<const i32x4_*>(q + 1024));
      if (t == TN - 1 && kb + 1 < p.KB) load((kb + 1) & 1, kb + 1);
#pragma unroll
      for (int j = 0; j < TM; ++j) mma8(acc[j][t], a, sw[t], b[j], sx[j]);
    }
  }
  const int ngroups = p.NP / 64;
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int64_t m = m0 + 16 * (wm * TM + j) + r;
    if (m >= p.M) continue;
#pragma unroll
    for (int q = 0; q < TN / 4; ++q) {
      const int grp = (tile0 + wn * TN) / 4 + q;
      if (grp < ngroups) {
        const f32x4 v[4] = {acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
        finish_group<GATED>(p, m, grp, lane, v);
      }
    }
  }
}

template <int NT, int MT, int XK, bool GATED>
static void launch_few(const M8Params& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.NP / 16 / NT), (unsigned)((p.M + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((matmul8_few_kernel<NT, MT, XK, GATED>), grid, dim3(64 * kFewWaves), 0, s, p);
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
  if (x_dtype == M3S_DTYPE_BF16) return launch_few<4, 1, kRowsBf16, GATED>(p, s);
  if (x_dtype == M3S_DTYPE_F32) return launch_few<4, 1, kRowsF32, GATED>(p, s);
  if (p.M <= 16) return launch_few<4, 1, kRows8, GATED>(p, s);
  if (p.M <= 256) return launch_few<4, 2, kRows8, GATED>(p, s);
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
  M3S_REQUIRE(!floats || a->ldx >= a->k, "m3s_matmul8: ldx is too short");
  M3S_REQUIRE(!a->residual || a->ldres >= a->n, "m3s_matmul8: ldres is too short");
  M3S_REQUIRE(a->gated || a->ldy >= a->n, "m3s_matmul8: ldy is too short");
  M8Params p{};
  p.x = a->x; p.xs = static_cast<const uint8_t*>(a->x_scales);
  p.w = static_cast<const uint8_t*>(a->w); p.ws = static_cast<const uint8_t*>(a->w_scales);
  p.bias = a->bias; p.residual = static_cast<const bf16*>(a->residual); p.y = static_cast<bf16*>(a->y);
  p.yv = static_cast<uint8_t*>(a->y_values); p.ys = static_cast<uint8_t*>(a->y_scales);
  p.M = a->rows; p.ldx = a->ldx; p.ldr = a->ldres; p.ldy = a->ldy;
  p.K = a->k; p.KB = (int)(padded8(a->k) / kStep8); p.N = a->n; p.act = a->activation;
  p.NP = (int)(a->gated ? 2 * padded8(a->n) : ((int64_t)a->n + 63) / 64 * 64);
  // scales are read through 32-bit offsets, and a launch holds at most 2^31 workgroups' tiles
  M3S_REQUIRE((int64_t)p.KB * p.M * 4 < (1ll << 31) && (int64_t)p.KB * p.NP * 4 < (1ll << 31),
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
