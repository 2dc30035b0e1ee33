// What is read off a language model's logits on gfx950: log-probabilities of given tokens with the
// entropy and the best alternatives, and the distillation loss from a teacher's best tokens, each
// with the gradient of the logits.
//
// For a row x of V logits at temperature T, with m = max x, d = x - m and s = sum e^{d / T}:
//
//   log p_j = d_j / T - log s,      H = log s - (sum e^{d / T} d) / (T s),
//   top: the k largest x, ties to the lower index;
//   dx_j = 1/T [ g_t (1[j = t] - p_j) - g_H p_j (log p_j + H) + sum_i g_i (1[j = id_i] - p_j) ].
//
// With a teacher's K tokens and logits u, w = softmax(u / T) over the K and q = softmax(x / T):
//
//   kd = T^2 sum_i w_i (log w_i - log q_{id_i}),     dx_j = T g (q_j - sum_{i: id_i = j} w_i),
//   nll = -log softmax(x)_t in the same pass,        dx_j += g_n (softmax(x)_j - 1[j = t]).
//
// The forward is one pass over the row with a running maximum; the sums kept are relative to it
// and rescaled when it grows. The gradient needs the finished sums, so it reads the row again and
// writes it once: both are bound by HBM. Row sums are float32; nothing but dlogits is rounded to
// the logits' type. p is formed as e^{d / T} / s from m and s (not from their combination
// m + log s, whose rounding would shift a whole row of p).
//
// Rows may start at any element: 16-byte accesses need no alignment on gfx950.
//
// Measured (us; TB/s of logits read and gradients written): log-probability and entropy of 8192 x
// 32000 float32, a tenth of it padding, forward 166 (5.7), backward 312 (6.4); distillation of 8192 x
// 50001 float32 with 32 teacher tokens and the cross-entropy, forward 253 (5.8), backward 497 (6.3);
// of 2048 x 65536 bf16, 53 (5.0) and 86 (6.3). A large copy moves 5.0 TB/s. 32768 x 256 float32, 16
// teacher tokens: 9.6 and 18.2, what is done once a row (sums over lanes, logarithms, the entries)
// taking half of it.
#include <algorithm>
#include <type_traits>

#include "m3s_common.h"
#include "m3s_internal.h"

namespace m3s {

constexpr int kRowThreads = 256;
constexpr int kTopMax = 64;        // alternatives of a row
constexpr int kTeacherMax = 256;   // teacher tokens of a row
// The threads to a row, by measurement (us, forward / backward of the distillation with 16 teacher
// tokens and a target, float32): many short rows go to 16 lanes each, as what is done once a row
// then costs a quarter (20971 x 400: 10.1 / 19.4 against 18.1 / 20.5 by a wave, 8192 x 1000: 8.7 / 16.6
// against 9.8 / 15.4; but 2048 x 1000: 5.3 / 6.5 against 4.6 / 5.8); rows up to 1024, and many up to
// 4096, to a wave (2048 x 1000: 4.6 / 5.8 against 6.2 / 9.7 by a workgroup, 4096 x 2000: 8.8 / 14.5
// against 12.5 / 14.9; but 512 x 4000: 5.4 / 5.8 against 4.7 / 5.8); the rest to a workgroup.
constexpr int kPartVocab = 1024, kPartRows = 4096, kWaveVocab = 4096, kWaveRows = 1024;
constexpr int kWaveHeld = 1024;     // one batch of a wave holds the row: it goes to one whatever the rows
constexpr int kPartTop = 24, kPartLanes = 8;        // alternatives that 16 lanes pick, of rows up to kPartPick long
constexpr int kPartPick = 256;
constexpr int kPartTeacher = 64;    // teacher tokens of a row of 16 lanes
constexpr float kNegInf = -__builtin_inff();

typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef bf16x8 bf16x8_any __attribute__((aligned(2)));

template <typename T> struct Piece;   // 16 bytes of a row
template <> struct Piece<float> {
  static constexpr int N = 4;
  __device__ static __forceinline__ void load(const float* p, float* x) {
    const f32x4 v = *reinterpret_cast<const f32x4_any*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v[i];
  }
  __device__ static __forceinline__ void store(float* p, const float* x) {
    *reinterpret_cast<f32x4_any*>(p) = f32x4{x[0], x[1], x[2], x[3]};
  }
};
template <> struct Piece<bf16> {
  static constexpr int N = 8;
  __device__ static __forceinline__ void load(const bf16* p, float* x) {
    const bf16x8 v = *reinterpret_cast<const bf16x8_any*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
  }
  __device__ static __forceinline__ void store(bf16* p, const float* x) {
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (bf16)x[i];
    *reinterpret_cast<bf16x8_any*>(p) = v;
  }
};

// ---- a row's group of lanes -------------------------------------------------------------------
// NT threads share a row: the workgroup, a wave, or 16 lanes (a row of the DPP moves) of a wave,
// which then handles four rows at once: what is done once a row (sums over lanes, logarithms,
// divisions) is what a short row costs.
template <int NT_>
struct Group {
  static constexpr int NT = NT_;
  static constexpr int NW = NT / 64;                    // waves; 0 for a part of one
  static constexpr int ROWS = kRowThreads / NT;         // rows to a workgroup
  static constexpr int TMP = NW == 4 ? 8 : 1;           // floats that the reductions need in LDS
  static __device__ __forceinline__ int tid() { return (int)threadIdx.x & (NT - 1); }
  // the group's place in the workgroup: wave-uniform for a wave, so that a row's scalars are scalar loads
  static __device__ __forceinline__ int slot() {
    if constexpr (NW == 4) return 0;
    const int s = (int)threadIdx.x / NT;
    return NW == 1 ? __builtin_amdgcn_readfirstlane(s) : s;
  }
  // what the group wrote to LDS or memory before is seen by it after
  static __device__ __forceinline__ void sync() {
    if constexpr (NW == 4) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
  // Reductions: the same value to every thread; `tmp` (TMP floats) is free afterwards.
  static __device__ __forceinline__ float max(float v, float* tmp) {
    v = fmaxf(v, dpp_mov<kDppQuadSwap1>(v));
    v = fmaxf(v, dpp_mov<kDppQuadSwap2>(v));
    v = fmaxf(v, dpp_mov<kDppHalfMirror>(v));
    v = fmaxf(v, dpp_mov<kDppRowMirror>(v));
    if constexpr (NW == 0) return v;
    const int i = __builtin_bit_cast(int, v);
    const auto row = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(i, l)); };
    v = fmaxf(fmaxf(row(0), row(16)), fmaxf(row(32), row(48)));
    if constexpr (NW == 4) {
      if (lane_id() == 0) tmp[threadIdx.x >> 6] = v;
      __syncthreads();
      v = fmaxf(fmaxf(tmp[0], tmp[1]), fmaxf(tmp[2], tmp[3]));
      __syncthreads();
    }
    return v;
  }
  static __device__ __forceinline__ void sum2(float& a, float& b, float* tmp) {
    if constexpr (NW == 0) {
      a = group_sum<16>(a);
      b = group_sum<16>(b);
      return;
    }
    a = wave_total(a);
    b = wave_total(b);
    if constexpr (NW == 4) {
      if (lane_id() == 0) {
        tmp[threadIdx.x >> 6] = a;
        tmp[4 + (threadIdx.x >> 6)] = b;
      }
      __syncthreads();
      a = (tmp[0] + tmp[1]) + (tmp[2] + tmp[3]);
      b = (tmp[4] + tmp[5]) + (tmp[6] + tmp[7]);
      __syncthreads();
    }
  }
  static __device__ __forceinline__ float sum(float v, float* tmp) {
    if constexpr (NW == 0) return group_sum<16>(v);
    v = wave_total(v);
    if constexpr (NW == 4) {
      if (lane_id() == 0) tmp[threadIdx.x >> 6] = v;
      __syncthreads();
      v = (tmp[0] + tmp[1]) + (tmp[2] + tmp[3]);
      __syncthreads();
    }
    return v;
  }
};

// ---- running sums of a row ------------------------------------------------------------------
// s = sum 2^{c (x - m)}, t = sum of the same times (x - m), s1 = sum 2^{c1 (x - m)}. A row of -inf
// keeps m = -inf and zeros; a NaN or +inf makes the sums NaN (fmaxf drops the NaN, s does not).
enum { kSingle = 0, kEntropy = 1, kDual = 2 };
// 2^{a b} with the product's rounding made good: a factor on a whole sum, so its error does not
// average out as the terms' do (one row of 131072 in pieces: log-probability off by 1e-7, not 5e-7).
__device__ __forceinline__ float exp2_product(float a, float b) {
  const float hi = a * b;
  return __builtin_amdgcn_exp2f(hi) * fmaf(fmaf(a, b, -hi), kLn2, 1.f);
}
template <int MODE>
struct RowSums {
  float m = kNegInf, s = 0.f, t = 0.f, s1 = 0.f;

  // m grows to at least `to`; the sums follow
  __device__ __forceinline__ void raise(float to, float c, float c1) {
    const float mn = fmaxf(m, to);
    const float ref = mn == kNegInf ? 0.f : mn;
    const float gap = fmaxf(m - ref, -1e30f);   // 0 * -1e30, not 0 * -inf, while s = 0
    const float f = exp2_product(gap, c);
    if constexpr (MODE == kEntropy) t = (t + s * gap) * f;
    s *= f;
    if constexpr (MODE == kDual) s1 *= exp2_product(gap, c1);
    m = mn;
  }
  // N more logits, the largest of them `top`. Their sums are formed first: one by one, the terms of a
  // batch would each be rounded at the size of the sum so far, which a likely token makes large (the
  // gradient of the log-probabilities, 8192 x 32000 float32: 0.9 to 1.2e-7 off as a whole so, 5.6e-8 by
  // batches, in the same time).
  template <int N>
  __device__ __forceinline__ void add(const float* x, float top, float c, float c1) {
    raise(top, c, c1);
    const float ref = m == kNegInf ? 0.f : m;
    float bs = 0.f, bt = 0.f, bs1 = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = x[i] - ref;
      const float e = __builtin_amdgcn_exp2f(d * c);
      bs += e;
      if constexpr (MODE == kEntropy) bt += e * fmaxf(d, -1e30f);
      if constexpr (MODE == kDual) bs1 += __builtin_amdgcn_exp2f(d * c1);
    }
    s += bs;
    if constexpr (MODE == kEntropy) t += bt;
    if constexpr (MODE == kDual) s1 += bs1;
  }
  template <typename G>
  __device__ __forceinline__ void join(float c, float c1, float* tmp) {
    raise(G::max(m, tmp), c, c1);
    if constexpr (MODE == kEntropy) G::sum2(s, t, tmp);
    else if constexpr (MODE == kDual) G::sum2(s, s1, tmp);
    else s = G::sum(s, tmp);
  }
};

template <int ctrl>
__device__ __forceinline__ int dpp_int(int v) {
  return __builtin_amdgcn_mov_dpp(v, ctrl, 0xF, 0xF, false);
}

// Where a thread's best logits lie: the largest maxima of its batches (U pieces of 16 bytes), the
// first two with their batch, so that the alternatives are found without reading the row again.
// The rest that fills no piece is not among them.
struct Best {
  float m1 = kNegInf, m2 = kNegInf, m3 = kNegInf;
  int b1 = -1, b2 = -1;   // -1: none seen, or none above -inf
  __device__ __forceinline__ void see(float v, int batch) {
    const bool first = v > m1, second = v > m2;
    m3 = fmaxf(m3, fminf(m2, v));
    b2 = first ? b1 : second ? batch : b2;
    m2 = first ? m1 : fmaxf(m2, v);
    b1 = first ? batch : b1;
    m1 = fmaxf(m1, v);
  }
};

// A thread's batch of a row of n logits: pieces batch U NT + u NT + tid, u < U; past the last whole
// batch come the logits that fill no piece, one a thread. Missing ones are -inf.
template <typename G, int U, typename T>
struct Rows {
  static constexpr int N = Piece<T>::N, HOP = G::NT * U, LEN = U * N;
  static __device__ __forceinline__ int whole(int n) { return (n / N + HOP - 1) / HOP; }   // batches
  static __device__ __forceinline__ int place(int batch, int i) {   // index of its i-th logit
    return (batch * HOP + i / N * G::NT + G::tid()) * N + i % N;
  }
  static __device__ __forceinline__ void load(const T* __restrict__ x, int n, int batch, float* v) {
    const int full = n / N, p = batch * HOP;
    if (p + HOP <= full) {
#pragma unroll
      for (int u = 0; u < U; ++u) Piece<T>::load(x + (int64_t)(p + u * G::NT + G::tid()) * N, v + u * N);
      return;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = p + u * G::NT + G::tid();
      if (at < full) {
        Piece<T>::load(x + (int64_t)at * N, v + u * N);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[u * N + i] = kNegInf;
      }
    }
  }
};

// The sums of a batch that may be the row's last, only of the pieces that it has; its largest logit.
template <typename G, int U, int MODE, typename T>
__device__ __forceinline__ float last_batch(RowSums<MODE>& r, const float* v, int n, int batch, float c,
                                            float c1) {
  using R = Rows<G, U, T>;
  const int full = n / R::N;
  float most = kNegInf;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (batch * R::HOP + u * G::NT >= full) break;
    float top = v[u * R::N];
#pragma unroll
    for (int i = 1; i < R::N; ++i) top = fmaxf(top, v[u * R::N + i]);
    most = fmaxf(most, top);
    r.template add<R::N>(v + u * R::N, top, c, c1);
  }
  return most;
}

// One pass over n logits by the group.
template <typename G, int U, bool TOP, int MODE, typename T>
__device__ __forceinline__ void row_pass(RowSums<MODE>& r, Best& best, const T* __restrict__ x, int n,
                                         float c, float c1) {
  using R = Rows<G, U, T>;
  const int full = n / R::N, batches = full / R::HOP;   // whole ones
  for (int b = 0; b < batches; ++b) {
    float v[R::LEN];
    R::load(x, n, b, v);
    float top = v[0];
#pragma unroll
    for (int i = 1; i < R::LEN; ++i) top = fmaxf(top, v[i]);
    if constexpr (TOP) best.see(top, b);
    r.template add<R::LEN>(v, top, c, c1);
  }
  if (batches * R::HOP < full) {
    float v[R::LEN];
    R::load(x, n, batches, v);
    const float most = last_batch<G, U, MODE, T>(r, v, n, batches, c, c1);
    if constexpr (TOP) best.see(most, batches);
  }
  const int at = n / R::N * R::N + G::tid();
  if (at < n) {
    const float v = (float)x[at];
    r.template add<1>(&v, v, c, c1);
  }
}

// A row of one batch and a rest, held: v[U N] is what fills no piece. Missing ones are -inf. Its sums.
template <typename G, int U, int MODE, typename T>
__device__ __forceinline__ void hold_row(RowSums<MODE>& r, float* v, const T* __restrict__ x, int n, float c,
                                         float c1) {
  using R = Rows<G, U, T>;
  const int tail = n / R::N * R::N + G::tid();
  R::load(x, n, 0, v);
  v[R::LEN] = tail < n ? (float)x[tail] : kNegInf;
  last_batch<G, U, MODE, T>(r, v, n, 0, c, c1);
  if (tail < n) r.template add<1>(v + R::LEN, v[R::LEN], c, c1);
}

// The workgroup's number. One row, or chunk of it, to each group and no loop over rows: a loop costs
// the kernels with alternatives 25 to 45 registers (46 without, eight waves a SIMD, 82 with, five).
__device__ __forceinline__ int64_t row_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// a / b for a >= 0 and b > 0, without the 64-bit division's hundred instructions where it can be.
__device__ __forceinline__ int64_t quotient(int64_t a, int b) {
  if (a < b) return 0;
  if (a >> 32 == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

template <typename T>
__device__ __forceinline__ const T* row_at(const m3s_blx& b, int64_t r, int seqlen) {
  const int64_t i = quotient(r, seqlen);
  return static_cast<const T*>(b.ptr) + i * b.stride_b + (r - i * seqlen) * b.stride_t;
}

// ---- the k largest of a row --------------------------------------------------------------------
// Unsigned keys in the floats' order (-0 counts as 0).
__device__ __forceinline__ uint32_t float_key(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_float(uint32_t k) {
  return __builtin_bit_cast(float, k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t kKeyMin = 0x007fffffu;   // the key of -inf

// A bound that at least k of the wave's 64 N values reach and no more than `most` >= k do, if ties
// allow it: found by ballots, first in doubling steps down from the largest value's key `top`,
// which the logits worth listing lie close to, then by halving. Of ties, the bound is the k-th value.
// Keys lose the bits that all of them share: bf16's lower 16, zeros or, below zero, ones.
template <typename T, int N>
__device__ __forceinline__ float kth_bound(const float* v, float top, int k, int most) {
  constexpr int SHIFT = sizeof(T) == 2 ? 16 : 0;
  constexpr uint32_t FIRST = kKeyMin >> SHIFT;
  const auto value = [](uint32_t key) {
    const bool below = !(key >> (31 - SHIFT));
    return key_float(key << SHIFT | (SHIFT && below ? 0xffffu : 0u));
  };
  uint32_t key[N];
#pragma unroll
  for (int i = 0; i < N; ++i) key[i] = float_key(v[i]) >> SHIFT;
  const auto reach = [&](uint32_t bar) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += __popcll(__ballot(key[i] >= bar));
    return n;
  };
  const uint32_t kt = __builtin_amdgcn_readfirstlane(float_key(top) >> SHIFT);
  uint32_t lo = FIRST, hi = kt + 1;   // at least k reach lo, fewer than k reach hi
  for (int j = 20 - SHIFT; j < 32 - SHIFT; ++j) {
    const uint32_t bar = kt - FIRST > (1u << j) ? kt - (1u << j) : FIRST;
    const int n = reach(bar);
    if (n >= k) {
      lo = bar;
      if (n <= most) return value(lo);
      break;
    }
    hi = bar;
  }
  while (hi - lo > 1) {
    const uint32_t bar = lo + (hi - lo) / 2;
    const int n = reach(bar);
    if (n >= k) {
      lo = bar;
      if (n <= most) break;
    } else {
      hi = bar;
    }
  }
  return value(lo);
}

// Inclusive prefix sum over a wave's lanes: within the rows of 16, then their totals.
__device__ __forceinline__ int wave_prefix(int v) {
  const int p = (int)row_prefix16((float)v);   // exact: small
  const int a = __builtin_amdgcn_readlane(p, 15), b = __builtin_amdgcn_readlane(p, 31);
  const int c = __builtin_amdgcn_readlane(p, 47), row = lane_id() >> 4;
  return p + (row > 0 ? a : 0) + (row > 1 ? b : 0) + (row > 2 ? c : 0);
}

// Candidates: (value, index) as one number, the better ones larger.
__device__ __forceinline__ uint64_t candidate(float v, int i) {
  return (uint64_t)float_key(v) << 32 | (uint32_t)~i;
}
template <int NW>
struct PickSpace {
  static constexpr int CAP = NW == 4 ? 1024 : 512, ITEMS = NW == 4 ? 512 : 1, WIDE = NW == 4 ? 256 : 1;
  uint64_t list[CAP + 4];
  float best[64 * NW];
  uint32_t item[ITEMS];   // thread and batch of a thread's best logits
  int wide[WIDE];         // threads whose other batches hold some too
  int count, items, wides, counts[4];
  float bar, tmp[8];
};
template <bool STRICT>
__device__ __forceinline__ bool reaches(float v, float bar) { return STRICT ? v > bar : v >= bar; }

template <int NW>
__device__ __forceinline__ void append(PickSpace<NW>& sp, float v, int i) {
  const int at = atomicAdd(&sp.count, 1);
  if (at < PickSpace<NW>::CAP) sp.list[at] = candidate(v, i);
}

// By a workgroup: lists every logit that reaches `bar`. The threads name the batches that hold one,
// then all of them read those, a piece of 16 bytes each. Returns the number, which may be more than
// the list holds (it is then cut short).
template <typename G, int U, bool STRICT, typename T>
__device__ __forceinline__ int gather(const T* __restrict__ x, int n, const Best& best, float bar,
                                      PickSpace<4>& sp) {
  using R = Rows<G, U, T>;
  constexpr int N = R::N;
  const int tid = G::tid(), full = n / N;
  if (tid == 0) sp.count = sp.items = sp.wides = 0;
  __syncthreads();
  if (reaches<STRICT>(best.m3, bar)) {
    sp.wide[atomicAdd(&sp.wides, 1)] = tid;
  } else if (reaches<STRICT>(best.m1, bar)) {   // above m3, so b1, and below b2, name a batch
    sp.item[atomicAdd(&sp.items, 1)] = (uint32_t)best.b1 << 8 | tid;
    if (reaches<STRICT>(best.m2, bar)) sp.item[atomicAdd(&sp.items, 1)] = (uint32_t)best.b2 << 8 | tid;
  }
  const int tail = full * N + tid;
  if (tail < n) {
    const float v = (float)x[tail];
    if (reaches<STRICT>(v, bar)) append(sp, v, tail);
  }
  __syncthreads();
  const auto piece = [&](int at) {   // by all lanes of the wave, past the row with nothing
    float v[N];
    uint32_t hits = 0;
    if (at < full) {
      Piece<T>::load(x + (int64_t)at * N, v);
#pragma unroll
      for (int i = 0; i < N; ++i) hits |= reaches<STRICT>(v[i], bar) ? 1u << i : 0u;
    }
    const int mine = __popc(hits), upto = wave_prefix(mine), all = __builtin_amdgcn_readlane(upto, 63);
    if (all == 0) return;
    int to = lane_id() == 0 ? atomicAdd(&sp.count, all) : 0;
    to = __builtin_amdgcn_readfirstlane(to) + upto - mine;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!(hits >> i & 1)) continue;
      if (to < PickSpace<4>::CAP) sp.list[to] = candidate(v[i], at * N + i);
      ++to;
    }
  };
  const int items = sp.items * U, wides = sp.wides;
  for (int q0 = 0; q0 < items; q0 += G::NT) {
    const int q = q0 + tid;
    const uint32_t it = q < items ? sp.item[q / U] : 0;
    piece(q < items ? (int)(it >> 8) * R::HOP + q % U * G::NT + (int)(it & 255) : full);
  }
  for (int w = 0; w < wides && *(volatile int*)&sp.count <= PickSpace<4>::CAP; ++w) {
    for (int at = sp.wide[w]; at < full; at += G::NT * G::NT) piece(at + tid * G::NT);
  }
  __syncthreads();
  return sp.count;
}

// Ranks the `count` listed candidates; those under k go out.
template <typename G, int NW, typename OUT>
__device__ __forceinline__ void rank_out(int count, int k, PickSpace<NW>& sp, OUT&& out) {
  if (G::tid() < 4) sp.list[count + G::tid()] = 0;   // below every candidate
  G::sync();
  for (int c = G::tid(); c < count; c += G::NT) {
    const uint64_t me = sp.list[c];
    int rank = 0;
    for (int j = 0; j < count; j += 4) {
#pragma unroll
      for (int u = 0; u < 4; ++u) rank += sp.list[j + u] > me;
    }
    if (rank < k) out(rank, key_float((uint32_t)(me >> 32)), (int)~(uint32_t)me);
  }
}

// Logits equal to `v`, in the order of their index, to the places from `from` up to k.
template <typename G, int NW, typename T, typename OUT>
__device__ __forceinline__ void equal_out(const T* __restrict__ x, int n, float v, int from, int k,
                                          PickSpace<NW>& sp, OUT&& out) {
  const int lane = lane_id();
  for (int p = 0; p < n && from < k; p += G::NT) {
    const int at = p + G::tid();
    const bool eq = at < n && (float)x[at] == v;
    const uint64_t m = __ballot(eq);
    int before = __popcll(m & ((1ull << lane) - 1)), all = __popcll(m);
    if constexpr (NW == 4) {
      const int wave = threadIdx.x >> 6;
      if (lane == 0) sp.counts[wave] = all;
      __syncthreads();
      all = 0;
      for (int w = 0; w < 4; ++w) {
        if (w < wave) before += sp.counts[w];
        all += sp.counts[w];
      }
      __syncthreads();
    }
    if (eq && from + before < k) out(from + before, v, at);
    from += all;
  }
}

// One value after another, for rows whose best logits all fell to few threads: the largest value
// below the last, then all that equal it.
template <typename G, int NW, typename T, typename OUT>
__device__ __forceinline__ void values_out(const T* __restrict__ x, int n, int k, PickSpace<NW>& sp,
                                           OUT&& out) {
  float last = __builtin_inff();
  for (int done = 0; done < k;) {
    float v = kNegInf;
    int same = 0;
    for (int i = G::tid(); i < n; i += G::NT) {
      const float e = (float)x[i];
      if (e < last) {
        same = e > v ? 1 : same + (e == v);
        v = fmaxf(v, e);
      }
    }
    const float top = G::max(v, sp.tmp);
    same = (int)G::sum(v == top ? (float)same : 0.f, sp.tmp);   // exact below 2^24, and k is 64
    equal_out<G>(x, n, top, done, k, sp, out);
    done += same;
    last = top;
    if (same == 0) break;
  }
}

// out(rank, value, index) for the k largest of n logits (k <= n, no NaN, no +inf, the largest
// `top`), equal ones by index. By a workgroup: a bound that k of the threads' maxima reach is reached
// by at least k logits, and by hardly more; those are collected from the few batches that hold them
// and ranked against each other. 999 rows of 50001 bf16 take 20 us, with 1, 20 and 64 alternatives
// 24, 25 and 28 (27, 43 and 53 with the exact k-th maximum, found bit by bit, and each thread reading
// its own batches; 5 ms by rounds of arg-max for 64).
template <typename G, int U, typename T, typename OUT>
__device__ __forceinline__ void pick(const T* __restrict__ x, int n, int k, float top, const Best& best,
                                     PickSpace<4>& sp, OUT&& out) {
  constexpr int CAP = PickSpace<4>::CAP;
  sp.best[threadIdx.x] = best.m1;
  __syncthreads();
  if (threadIdx.x < 64) {
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = sp.best[64 * i + threadIdx.x];
    const float bar = kth_bound<T, 4>(m, top, k, min(k + 12, 64));
    if (threadIdx.x == 0) sp.bar = bar;
  }
  __syncthreads();
  const float bar = sp.bar;
  int count = gather<G, U, false>(x, n, best, bar, sp);
  if (count > CAP) {   // many ties, as in masked rows: what exceeds them, then the first of them
    __syncthreads();
    count = gather<G, U, true>(x, n, best, bar, sp);
    if (count > CAP) {
      values_out<G>(x, n, k, sp, out);
      return;
    }
    equal_out<G>(x, n, bar, count, k, sp, out);
  }
  rank_out<G>(count, k, sp, out);
  __syncthreads();   // the space is free again
}

// The same by a wave that holds the whole row, one batch and a rest. The bound is on the lanes'
// maxima for few alternatives (one value a lane to count), on the logits themselves for more, of
// which the lanes' maxima would let most of the row through. 8192 x 512 float32 takes 3.7 us, with 1,
// 20 and 64 alternatives 7.4, 9.3 and 19. (When 20 took 11.9 so, listing by ballots logit for logit took
// 12.5, and an atomic for each logit with the row read again 14.8.)
template <typename G, int U, typename T, typename OUT>
__device__ __forceinline__ void pick_held(const T* __restrict__ x, const float* v, int n, int k, float top,
                                          PickSpace<1>& sp, OUT&& out) {
  using R = Rows<G, U, T>;
  constexpr int LEN = R::LEN;
  // so many lanes' logits all fit the list: no bound lets more of them through but by ties, and
  // what exceeds the tied value then comes from fewer than k lanes
  constexpr int LANES = std::min(64, PickSpace<1>::CAP / (LEN + 1)), FEW = std::min(24, LANES);
  const int whole = n / R::N * R::N, tail = whole + G::tid();
  float bar;
  if (k <= min(FEW, n / R::N / 2)) {   // at most half of the lanes that hold something
    float most = v[0];
#pragma unroll
    for (int i = 1; i <= LEN; ++i) most = fmaxf(most, v[i]);
    bar = kth_bound<T, 1>(&most, top, k, min(k + 12, LANES));
  } else {
    bar = kth_bound<T, LEN + 1>(v, top, k, 64);
  }
  const auto gather = [&](auto strict) {
    constexpr bool STRICT = decltype(strict)::value;
    uint32_t hits = 0;
#pragma unroll
    for (int i = 0; i <= LEN; ++i) hits |= reaches<STRICT>(v[i], bar) ? 1u << i : 0u;
    if (bar == kNegInf) {   // where there is no logit stands -inf too
#pragma unroll
      for (int i = 0; i < LEN; ++i) hits &= R::place(0, i) < whole ? ~0u : ~(1u << i);
      hits &= tail < n ? ~0u : ~(1u << LEN);
    }
    const int mine = __popc(hits), upto = wave_prefix(mine), all = __builtin_amdgcn_readlane(upto, 63);
    int at = upto - mine;
    if (all <= PickSpace<1>::CAP) {
      for (; hits; hits &= hits - 1) {   // read again: few, and no register has a running index
        const int i = __builtin_ctz(hits), where = i < LEN ? R::place(0, i) : tail;
        sp.list[at++] = candidate((float)x[where], where);
      }
    }
    G::sync();
    return all;
  };
  int count = gather(std::false_type());
  if (count > PickSpace<1>::CAP) {
    G::sync();
    count = gather(std::true_type());   // fewer than FEW (LEN + 1), or than k
    equal_out<G>(x, n, bar, count, k, sp, out);
  }
  rank_out<G>(count, k, sp, out);
  G::sync();
}

// The same by 16 lanes that hold the row's at most kPartPick logits: the bound on the lanes' maxima by
// comparing each with the others, beyond kPartLanes alternatives on two maxima of each (of 16 values
// a k-th near the last lets most of the row through); the logits that reach it in a list, ranked. One,
// and a list too long or a bound of -inf (ties, masked rows, fewer maxima than alternatives), go by
// rounds of (largest value, lowest index). 32768 x 256 float32 takes 6 us, with 1, 5, 8, 14, 20 and 24
// alternatives 8.5, 10.7, 11.8, 14.8, 18.7 and 22.7 (in bf16 20 and 24 take 17.4 and 22.5); by rounds 5
// and 8 took 15 and 18.7, on one maximum of each lane 14 took 22, and by a wave 25 take 27 (bf16 31).
struct PartSpace {
  static constexpr int CAP = 96;
  uint64_t list[CAP + 5];   // four zeros behind it; odd: the groups use different banks
};
// f(turned) for each of a lane's 15 neighbours in 16: turned(v) is that lane's v.
template <int n = 1, typename F>
__device__ __forceinline__ void others(F&& f) {
  f([](float v) { return dpp_mov<0x120 + n>(v); });
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (n < 15) others<n + 1>(f);
}
template <typename G, int U, typename T, typename OUT>
__device__ __forceinline__ void pick_part(const T* __restrict__ x, float* v, int n, int k, PartSpace& sp,
                                          OUT&& out) {
  using R = Rows<G, U, T>;
  constexpr int N = R::N, LEN = R::LEN;
  const int whole = n / N * N, tail = whole + G::tid();
  if (k > 1) {
    float even = v[LEN], odd = kNegInf;   // a lane's largest of each kind
#pragma unroll
    for (int i = 0; i < LEN; i += 2) {
      even = fmaxf(even, v[i]);
      odd = fmaxf(odd, v[i + 1]);
    }
    float bar;   // the k-th largest of the lanes' maxima, or of both of each: the largest that k of them reach
    if (k <= kPartLanes) {
      const float most = fmaxf(even, odd);
      int reach = 1;
      others([&](auto turned) { reach += turned(most) >= most; });
      bar = reach >= k ? most : kNegInf;
    } else {
      int reach0 = 1 + (odd >= even), reach1 = 1 + (even >= odd);
      others([&](auto turned) {
        const float a = turned(even), b = turned(odd);
        reach0 += (a >= even) + (b >= even);
        reach1 += (a >= odd) + (b >= odd);
      });
      bar = fmaxf(reach0 >= k ? even : kNegInf, reach1 >= k ? odd : kNegInf);
    }
    bar = G::max(bar, nullptr);
    uint32_t hits = 0;
#pragma unroll
    for (int i = 0; i <= LEN; ++i) hits |= v[i] >= bar ? 1u << i : 0u;
    const float upto = row_prefix16((float)__popc(hits));
    const int total = (int)G::max(upto, nullptr);
    if (bar > kNegInf && total <= PartSpace::CAP) {   // -inf may be a logit or none
      int at = (int)upto - __popc(hits);
      for (; hits; hits &= hits - 1) {   // read again: few, and no register has a running index
        const int i = __builtin_ctz(hits), where = i < LEN ? R::place(0, i) : tail;
        sp.list[at++] = candidate((float)x[where], where);
      }
      if (G::tid() < 4) sp.list[total + G::tid()] = 0;   // below every candidate
      G::sync();
      for (int c = G::tid(); c < total; c += G::NT) {
        const uint64_t me = sp.list[c];
        int rank = 0;
        for (int j = 0; j < total; j += 4) {
#pragma unroll
          for (int u = 0; u < 4; ++u) rank += sp.list[j + u] > me;
        }
        if (rank < k) out(rank, key_float((uint32_t)(me >> 32)), (int)~(uint32_t)me);
      }
      G::sync();
      return;
    }
  }
  const float gone = __builtin_nanf("");   // no logit, or one that is out already
#pragma unroll
  for (int i = 0; i < LEN; ++i) v[i] = i / N * G::NT + G::tid() < n / N ? v[i] : gone;
  v[LEN] = tail < n ? v[LEN] : gone;
  for (int j = 0; j < k; ++j) {
    float top = v[LEN];
#pragma unroll
    for (int i = 0; i < LEN; ++i) top = fmaxf(top, v[i]);
    top = G::max(top, nullptr);
    int own = LEN + 1;   // a lane's places rise with i
#pragma unroll
    for (int i = LEN; i >= 0; --i) own = v[i] == top ? i : own;
    const int mine = own > LEN ? 0x7fffffff : own < LEN ? R::place(0, own) : tail;
    int at = mine;
    at = min(at, dpp_int<kDppQuadSwap1>(at));
    at = min(at, dpp_int<kDppQuadSwap2>(at));
    at = min(at, dpp_int<kDppHalfMirror>(at));
    at = min(at, dpp_int<kDppRowMirror>(at));
    own = mine == at ? own : -1;
#pragma unroll
    for (int i = 0; i <= LEN; ++i) v[i] = i == own ? gone : v[i];
    if (G::tid() == (j & 15)) out(j, top, at);
  }
}

// ---- log-probabilities ----------------------------------------------------------------------
struct LogprobParams {
  m3s_blx logits;
  const int64_t* targets;
  float *logp, *entropy, *stats, *top_logp;
  int64_t* top_ids;
  const float *dlogp, *dentropy, *dtop;
  void* dlogits;
  float* part;       // a split row's pieces: (rows, split, 3) sums, (rows, split, top) values and ids
  int64_t ignore, rows;
  int seqlen, vocab, top, chunks, chunk, split, share;   // chunk, share: logits to one of chunks, to a piece
  float inv_t, c;
};

struct LogprobParts {
  float *sums, *v;
  int* i;
  __device__ LogprobParts(const LogprobParams& p, int64_t r) {
    const int64_t all = p.rows * p.split;
    sums = p.part + 3 * r * p.split;
    v = p.part + 3 * all + r * p.split * p.top;
    i = reinterpret_cast<int*>(p.part + (3 + p.top) * all) + r * p.split * p.top;
  }
};

// A row without a token at it: the logits are not read.
template <typename G>
__device__ __forceinline__ void logprob_skip(const LogprobParams& p, int64_t r) {
  if (G::tid() == 0) {
    p.logp[r] = p.entropy[r] = 0.f;
    if (p.stats) p.stats[3 * r] = p.stats[3 * r + 1] = p.stats[3 * r + 2] = 0.f;
  }
  for (int j = G::tid(); j < p.top; j += G::NT) {
    p.top_logp[r * p.top + j] = kNegInf;
    p.top_ids[r * p.top + j] = -1;
  }
}

struct LogprobRow {   // from finished sums
  float m, logs, inv_t;
  bool empty;
  __device__ LogprobRow(const RowSums<kEntropy>& s, float inv_t_)
      : m(s.m), logs(logf(s.s)), inv_t(inv_t_), empty(s.m == kNegInf && s.s == 0.f) {}
  __device__ float operator()(float v) const { return empty ? kNegInf : (v - m) * inv_t - logs; }
};

// The target's logit (NaN where there is none), loaded ahead of the row.
template <typename T>
__device__ __forceinline__ float target_logit(const LogprobParams& p, int64_t tgt, const T* x) {
  return p.targets && tgt >= 0 && tgt < p.vocab ? (float)x[tgt] : __builtin_nanf("");
}

template <typename G>
__device__ __forceinline__ void logprob_store(const LogprobParams& p, int64_t r, int64_t tgt, float xt,
                                              const RowSums<kEntropy>& sum, const LogprobRow& logp) {
  if (G::tid() != 0) return;
  const float h = logp.empty ? 0.f : logp.logs - sum.t * p.inv_t / sum.s;
  p.entropy[r] = h;
  if (p.stats) {
    p.stats[3 * r] = sum.m;
    p.stats[3 * r + 1] = sum.s;
    p.stats[3 * r + 2] = h;
  }
  if (p.targets) p.logp[r] = tgt >= 0 && tgt < p.vocab ? logp(xt) : __builtin_nanf("");
}

// NaN or +inf among the logits: no order to report.
template <typename G>
__device__ __forceinline__ void logprob_unordered(const LogprobParams& p, int64_t r) {
  for (int j = G::tid(); j < p.top; j += G::NT) {
    p.top_logp[r * p.top + j] = __builtin_nanf("");
    p.top_ids[r * p.top + j] = -1;
  }
}

template <bool TOP, int NT, int U, typename T>
__global__ void __launch_bounds__(kRowThreads) logprob_fwd_kernel(const LogprobParams p) {
  using G = Group<NT>;
  constexpr bool HELD = TOP && NT < 256;   // the row stays in registers between its sums and the pick
  __shared__ float tmp[G::TMP];
  __shared__ std::conditional_t<NT == 16, PartSpace, PickSpace<NT == 256 ? 4 : 1>> space[TOP ? G::ROWS : 1];
  const int64_t r = row_block() * G::ROWS + G::slot();
  if (r >= p.rows) return;
  const int64_t tgt = p.targets ? p.targets[r] : 0;
  if (p.targets && tgt == p.ignore) {
    logprob_skip<G>(p, r);
    return;
  }
  const T* x = row_at<T>(p.logits, r, p.seqlen);
  const float xt = target_logit(p, tgt, x);
  RowSums<kEntropy> sum;
  Best best;
  float held[HELD ? U * Piece<T>::N + 1 : 1];
  if constexpr (HELD) hold_row<G, U>(sum, held, x, p.vocab, p.c, 0.f);
  else row_pass<G, U, TOP>(sum, best, x, p.vocab, p.c, 0.f);
  sum.template join<G>(p.c, 0.f, tmp);
  const LogprobRow logp(sum, p.inv_t);
  logprob_store<G>(p, r, tgt, xt, sum, logp);
  if constexpr (TOP) {
    if (sum.s != sum.s) {
      logprob_unordered<G>(p, r);
      return;
    }
    const auto out = [&](int j, float v, int i) {
      p.top_logp[r * p.top + j] = logp(v);
      p.top_ids[r * p.top + j] = i;
    };
    if constexpr (NT == 256) pick<G, U>(x, p.vocab, p.top, sum.m, best, space[G::slot()], out);
    else if constexpr (NT == 64) pick_held<G, U>(x, held, p.vocab, p.top, sum.m, space[G::slot()], out);
    else pick_part<G, U>(x, held, p.vocab, p.top, space[G::slot()], out);
  }
}

// Few long rows: a workgroup to each of a row's `split` pieces ...
template <bool TOP, int U, typename T>
__global__ void __launch_bounds__(kRowThreads) logprob_piece_kernel(const LogprobParams p) {
  using G = Group<256>;
  __shared__ float tmp[G::TMP];
  __shared__ PickSpace<4> space[1];
  const int64_t r = blockIdx.x / p.split;
  const int g = (int)(blockIdx.x - r * p.split);
  if (p.targets && p.targets[r] == p.ignore) return;
  const int lo = g * p.share, n = min(p.share, p.vocab - lo);
  const T* x = row_at<T>(p.logits, r, p.seqlen) + lo;
  const LogprobParts part(p, r);
  RowSums<kEntropy> sum;
  Best best;
  row_pass<G, U, TOP>(sum, best, x, n, p.c, 0.f);
  sum.template join<G>(p.c, 0.f, tmp);
  if (threadIdx.x == 0) {
    part.sums[3 * g] = sum.m;
    part.sums[3 * g + 1] = sum.s;
    part.sums[3 * g + 2] = sum.t;
  }
  if constexpr (TOP) {
    float* pv = part.v + g * p.top;
    int* pi = part.i + g * p.top;
    const int k = sum.s != sum.s ? 0 : min(p.top, n);
    for (int j = k + threadIdx.x; j < p.top; j += kRowThreads) {   // never among the best of the row
      pv[j] = kNegInf;
      pi[j] = -1;
    }
    if (k) {
      pick<G, U>(x, n, k, sum.m, best, space[0], [&](int j, float v, int i) {
        pv[j] = v;
        pi[j] = lo + i;
      });
    }
  }
}

// ... and one to join them. Pieces stand in the order of the row and hold their best in order, so
// equal values are in the order of their index here too.
template <bool TOP, typename T>
__global__ void __launch_bounds__(kRowThreads) logprob_join_kernel(const LogprobParams p) {
  using G = Group<256>;
  __shared__ float tmp[G::TMP];
  __shared__ PickSpace<4> space[1];
  const int64_t r = blockIdx.x;
  const int64_t tgt = p.targets ? p.targets[r] : 0;
  if (p.targets && tgt == p.ignore) {
    logprob_skip<G>(p, r);
    return;
  }
  const float xt = target_logit(p, tgt, row_at<T>(p.logits, r, p.seqlen));
  const LogprobParts part(p, r);
  RowSums<kEntropy> sum;
  if ((int)threadIdx.x < p.split) {
    sum.m = part.sums[3 * threadIdx.x];
    sum.s = part.sums[3 * threadIdx.x + 1];
    sum.t = part.sums[3 * threadIdx.x + 2];
  }
  sum.template join<G>(p.c, 0.f, tmp);
  const LogprobRow logp(sum, p.inv_t);
  logprob_store<G>(p, r, tgt, xt, sum, logp);
  if constexpr (TOP) {
    if (sum.s != sum.s) {
      logprob_unordered<G>(p, r);
      return;
    }
    const int n = p.split * p.top;
    Best best;
    const int batches = Rows<G, 1, float>::whole(n);
    for (int b = 0; b < batches; ++b) {
      float v[4];
      Rows<G, 1, float>::load(part.v, n, b, v);
      best.see(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), b);
    }
    pick<G, 1>(part.v, n, p.top, sum.m, best, space[0], [&](int j, float v, int i) {
      p.top_logp[r * p.top + j] = logp(v);
      p.top_ids[r * p.top + j] = part.i[i];
    });
  }
}

// ---- gradients ---------------------------------------------------------------------------------
// The dense part: f(x) for every logit of lo .. hi - 1, at most kBwdPieces pieces a thread. At 8192 x
// 50001 the log-probabilities' backward takes 525 us in float32 (585 with two, 621 with three) and 298 in
// bf16 (272 and 291), the distillation's 527 (541 and 610) and 314 (323 and 311); at 65536 x 1000 float32,
// by 16 lanes, the latter takes 120 (176 and 144).
constexpr int kBwdPieces = 4;
// P pieces a thread, without a branch between them: past the last piece a thread takes that one again,
// and writes what its owner writes. (A wait behind a branch is for everything, stores too: one for each
// piece would wait for the piece before to reach memory.)
template <typename G, int P, typename T, typename F>
__device__ __forceinline__ void pieces_map(const T* __restrict__ x, T* __restrict__ dx, int full, F&& f) {
  constexpr int N = Piece<T>::N;
  float v[P * N];
#pragma unroll
  for (int u = 0; u < P; ++u) Piece<T>::load(x + min(u * G::NT + G::tid(), full - 1) * N, v + u * N);
#pragma unroll
  for (int u = 0; u < P; ++u) {
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = f(v[u * N + i]);
    Piece<T>::store(dx + min(u * G::NT + G::tid(), full - 1) * N, o);
  }
}
template <typename G, typename T, typename F>
__device__ __forceinline__ void chunk_map(const T* __restrict__ x, T* __restrict__ dx, int lo, int hi,
                                          F&& f) {
  constexpr int N = Piece<T>::N;
  const int n = hi - lo, full = n / N;
  static_assert(kBwdPieces == 4);   // the cases below
  if (full > 3 * G::NT) pieces_map<G, 4>(x + lo, dx + lo, full, f);
  else if (full > 2 * G::NT) pieces_map<G, 3>(x + lo, dx + lo, full, f);
  else if (full > G::NT) pieces_map<G, 2>(x + lo, dx + lo, full, f);
  else if (full > 0) pieces_map<G, 1>(x + lo, dx + lo, full, f);
  const int at = full * N + G::tid();
  if (at < n) dx[lo + at] = (T)f((float)x[lo + at]);
}
template <typename G, typename T>
__device__ __forceinline__ void chunk_zero(T* __restrict__ dx, int lo, int hi) {
  constexpr int N = Piece<T>::N;
  const float zero[N] = {};
  const int full = (hi - lo) / N;
  for (int at = G::tid(); at < full; at += G::NT) Piece<T>::store(dx + lo + at * N, zero);
  const int at = lo + full * N + G::tid();
  if (at < hi) dx[at] = (T)0.f;
}

template <int NT, typename T>
__global__ void __launch_bounds__(kRowThreads) logprob_bwd_kernel(const LogprobParams p) {
  using G = Group<NT>;
  __shared__ int sids[G::ROWS][kTopMax + 1];   // odd: the groups of a wave on different banks
  __shared__ float sgrad[G::ROWS][kTopMax + 1];
  int* ids = sids[G::slot()];
  float* gtop = sgrad[G::slot()];
  const int64_t w = row_block() * G::ROWS + G::slot();
  if (w >= p.rows * p.chunks) return;
  const int64_t r = quotient(w, p.chunks);
  const int lo = (int)(w - r * p.chunks) * p.chunk, hi = min(lo + p.chunk, p.vocab);
  const T* x = row_at<T>(p.logits, r, p.seqlen);
  T* dx = static_cast<T*>(p.dlogits) + r * p.vocab;
  const int64_t tgt = p.targets ? p.targets[r] : -1;
  const float m = p.stats[3 * r], s = p.stats[3 * r + 1], h = p.stats[3 * r + 2];
  // an ignored row, and one of nothing but -inf, has s = 0 and no gradient
  if (s == 0.f) {
    chunk_zero<G>(dx, lo, hi);
    return;
  }
  float gl = p.dlogp ? p.dlogp[r] * p.inv_t : 0.f;
  if (p.dlogp && (tgt < 0 || tgt >= p.vocab)) gl = __builtin_nanf("");
  const float gh = p.dentropy ? p.dentropy[r] * p.inv_t : 0.f;
  float g = gl;
  const int top = p.dtop ? p.top : 0;
  for (int j = 0; j < top; ++j) g += p.dtop[r * top + j] * p.inv_t;
  const float inv_s = 1.f / s, logs = logf(s);
  const auto f = [&](float v) {
    const float d = v - m;
    const float q = __builtin_amdgcn_exp2f(d * p.c) * inv_s;
    const float lq = fmaxf(d * p.inv_t - logs, -1e30f);
    return -q * (g + gh * (lq + h));
  };
  chunk_map<G>(x, dx, lo, hi, f);
  // then the entries that a token or an alternative adds to, whole
  for (int j = G::tid(); j < top; j += G::NT) {
    ids[j] = (int)p.top_ids[r * top + j];
    gtop[j] = p.dtop[r * top + j] * p.inv_t;
  }
  G::sync();
  for (int j = G::tid(); j < top; j += G::NT) {
    const int i = ids[j];
    if (i >= lo && i < hi) dx[i] = (T)(f((float)x[i]) + gtop[j] + (i == tgt ? gl : 0.f));
  }
  if (G::tid() == 0 && p.dlogp && tgt >= lo && tgt < hi) {
    bool alone = true;
    for (int j = 0; j < top; ++j) alone = alone && ids[j] != tgt;
    if (alone) dx[tgt] = (T)(f((float)x[tgt]) + gl);
  }
}

// ---- distillation ---------------------------------------------------------------------------
struct DistillParams {
  m3s_blx logits;
  const void *ids, *teacher;
  const int64_t* targets;
  float *kd, *nll, *stats;
  const float *dkd, *dnll;
  void* dlogits;
  float* part;       // a split row's pieces: (rows, split, 3) sums
  int64_t ignore, rows;
  int seqlen, vocab, k, chunks, chunk, id_bytes, teacher_bf16, split, share;
  float temp, inv_t, c, c1;
};

__device__ __forceinline__ int64_t teacher_id(const DistillParams& p, int64_t at) {
  return p.id_bytes == 8 ? static_cast<const int64_t*>(p.ids)[at] : (int64_t)static_cast<const int32_t*>(p.ids)[at];
}
__device__ __forceinline__ float teacher_logit(const DistillParams& p, int64_t at) {
  return p.teacher_bf16 ? (float)static_cast<const bf16*>(p.teacher)[at] : static_cast<const float*>(p.teacher)[at];
}

// A row's teacher tokens, kTeacherMax / NT to a thread: ids (-1: none, or outside the vocabulary),
// logits, and e^{(u - ref) / T}.
// ts = 0 says that there is no entry, NaN that one is a NaN or an id outside the vocabulary.
template <typename G>
struct Teacher {
  static constexpr int N = (G::NT == 16 ? kPartTeacher : kTeacherMax) / G::NT;
  int id[N];
  float u[N], e[N], ref, ts;
  __device__ __forceinline__ Teacher(const DistillParams& p, int64_t r, float* tmp) {
    float top = kNegInf, sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = i * G::NT + G::tid();
      id[i] = -1;
      u[i] = kNegInf;
      if (at < p.k) {
        const int64_t v = teacher_id(p, r * p.k + at);
        if (v >= 0) u[i] = v < p.vocab ? teacher_logit(p, r * p.k + at) : __builtin_nanf("");
        if (v >= 0 && v < p.vocab) id[i] = (int)v;
      }
      top = fmaxf(top, u[i]);
    }
    top = G::max(top, tmp);
    ref = top == kNegInf ? 0.f : top;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      e[i] = __builtin_amdgcn_exp2f((u[i] - ref) * p.c);
      sum += e[i];
    }
    ts = G::sum(sum, tmp);
  }
};

// From a row's finished sums: its losses and stats (rows, 5): m, sum e^{d / T}, sum e^d, the
// teacher's maximum and sum. A row with nothing to learn (its logits were not read) has zeros.
template <typename G, int MODE, typename T>
__device__ __forceinline__ void distill_store(const DistillParams& p, int64_t r, const T* x,
                                              const Teacher<G>& t, bool hard, int64_t tgt,
                                              const RowSums<MODE>& sum, float* tmp) {
  const bool soft = t.ts != 0.f, empty = sum.m == kNegInf && sum.s == 0.f;
  const float logs = logf(sum.s), logts = logf(t.ts), inv_ts = 1.f / t.ts;
  float term = 0.f;
#pragma unroll
  for (int i = 0; i < Teacher<G>::N; ++i) {
    if (t.e[i] == 0.f || !soft) continue;   // weight 0; NaN goes on
    const float lw = (t.u[i] - t.ref) * p.inv_t - logts;
    const float xi = t.id[i] >= 0 ? (float)x[t.id[i]] : __builtin_nanf("");
    const float lq = empty ? kNegInf : (xi - sum.m) * p.inv_t - logs;
    term += t.e[i] * inv_ts * (lw - lq);
  }
  const float kd = G::sum(term, tmp);
  if (G::tid() != 0) return;
  p.kd[r] = soft ? p.temp * p.temp * kd : 0.f;
  const float s1 = MODE == kDual ? sum.s1 : sum.s;
  if (p.stats) {
    float* stats = p.stats + 5 * r;
    stats[0] = soft || hard ? sum.m : 0.f;
    stats[1] = sum.s;
    stats[2] = s1;
    stats[3] = t.ref;
    stats[4] = t.ts;
  }
  if (p.nll) {
    float v = 0.f;
    if (hard) {
      v = tgt < 0 || tgt >= p.vocab ? __builtin_nanf("")
          : empty                   ? __builtin_inff()
                                    : logf(s1) - ((float)x[tgt] - sum.m);
    }
    p.nll[r] = v;
  }
}

// MODE kDual where the cross-entropy's sum is another than the teacher's, else kSingle.
template <int MODE, int NT, int U, typename T>
__global__ void __launch_bounds__(kRowThreads) distill_fwd_kernel(const DistillParams p) {
  using G = Group<NT>;
  __shared__ float tmp[G::TMP];
  const int64_t r = row_block() * G::ROWS + G::slot();
  if (r >= p.rows) return;
  const T* x = row_at<T>(p.logits, r, p.seqlen);
  const Teacher<G> t(p, r, tmp);
  const int64_t tgt = p.targets ? p.targets[r] : 0;
  const bool hard = p.targets && tgt != p.ignore;
  RowSums<MODE> sum;
  if (t.ts != 0.f || hard) {
    Best unused;
    row_pass<G, U, false>(sum, unused, x, p.vocab, p.c, p.c1);
    sum.template join<G>(p.c, p.c1, tmp);
  }
  distill_store<G>(p, r, x, t, hard, tgt, sum, tmp);
}

// Few long rows: a workgroup to each of a row's pieces, then one to join them.
template <int MODE, int U, typename T>
__global__ void __launch_bounds__(kRowThreads) distill_piece_kernel(const DistillParams p) {
  using G = Group<256>;
  __shared__ float tmp[G::TMP];
  const int64_t r = blockIdx.x / p.split;
  const int g = (int)(blockIdx.x - r * p.split);
  const int lo = g * p.share, n = min(p.share, p.vocab - lo);
  if (!p.targets || p.targets[r] == p.ignore) {   // without a teacher token either: not read
    bool any = false;
    for (int j = threadIdx.x; j < p.k; j += kRowThreads) any = any || teacher_id(p, r * p.k + j) >= 0;
    if (!__syncthreads_or(any)) return;
  }
  RowSums<MODE> sum;
  Best unused;
  row_pass<G, U, false>(sum, unused, row_at<T>(p.logits, r, p.seqlen) + lo, n, p.c, p.c1);
  sum.template join<G>(p.c, p.c1, tmp);
  if (threadIdx.x == 0) {
    float* out = p.part + 3 * (r * p.split + g);
    out[0] = sum.m;
    out[1] = sum.s;
    if (MODE == kDual) out[2] = sum.s1;
  }
}

template <int MODE, typename T>
__global__ void __launch_bounds__(kRowThreads) distill_join_kernel(const DistillParams p) {
  using G = Group<256>;
  __shared__ float tmp[G::TMP];
  const int64_t r = blockIdx.x;
  const Teacher<G> t(p, r, tmp);
  const int64_t tgt = p.targets ? p.targets[r] : 0;
  const bool hard = p.targets && tgt != p.ignore;
  RowSums<MODE> sum;
  if (t.ts != 0.f || hard) {
    if ((int)threadIdx.x < p.split) {
      const float* in = p.part + 3 * (r * p.split + threadIdx.x);
      sum.m = in[0];
      sum.s = in[1];
      if (MODE == kDual) sum.s1 = in[2];
    }
    sum.template join<G>(p.c, p.c1, tmp);
  }
  distill_store<G>(p, r, row_at<T>(p.logits, r, p.seqlen), t, hard, tgt, sum, tmp);
}

// DUAL: both losses, at two temperatures; else one exponential serves (kd alone or the
// cross-entropy alone at its own c, or both at temperature 1).
template <bool DUAL, int NT, typename T>
__global__ void __launch_bounds__(kRowThreads) distill_bwd_kernel(const DistillParams p) {
  using G = Group<NT>;
  constexpr int KMAX = NT == 16 ? kPartTeacher : kTeacherMax;
  __shared__ int sids[G::ROWS][KMAX + 1];   // odd: the groups of a wave on different banks
  __shared__ float sweight[G::ROWS][KMAX + 1];
  const int64_t w = row_block() * G::ROWS + G::slot();
  if (w >= p.rows * p.chunks) return;
  const int64_t r = quotient(w, p.chunks);
  const int lo = (int)(w - r * p.chunks) * p.chunk, hi = min(lo + p.chunk, p.vocab);
  const T* x = row_at<T>(p.logits, r, p.seqlen);
  T* dx = static_cast<T*>(p.dlogits) + r * p.vocab;
  const float* stats = p.stats + 5 * r;
  const float m = stats[0], s = stats[1], s1 = stats[2], ref = stats[3], ts = stats[4];
  const int64_t tgt = p.targets ? p.targets[r] : p.ignore;
  const bool soft = p.dkd && ts != 0.f, hard = p.dnll && tgt != p.ignore;
  if (s == 0.f || (!soft && !hard)) {   // no loss, or no distribution
    chunk_zero<G>(dx, lo, hi);
    return;
  }
  const float a = soft ? p.dkd[r] * p.temp : 0.f, as = ts != ts ? ts : a / s;
  float b = hard ? p.dnll[r] : 0.f;
  if (hard && (tgt < 0 || tgt >= p.vocab)) b = __builtin_nanf("");
  const float bs = b / s1;
  // one exponential: of the teacher's temperature, or of the cross-entropy's if it is alone
  const float ec = soft ? p.c : p.c1, es = soft ? (hard ? as + bs : as) : bs;
  const auto f = [&](float v) {
    const float d = v - m;
    if constexpr (!DUAL) return es * __builtin_amdgcn_exp2f(d * ec);
    float o = 0.f;
    if (soft) o = as * __builtin_amdgcn_exp2f(d * p.c);
    if (hard) o += bs * __builtin_amdgcn_exp2f(d * p.c1);
    return o;
  };
  const int k = soft ? p.k : 0;
  const float at = a / ts;
  const auto weight = [&](int64_t id, int j) {   // what an entry takes
    if (id < 0 || id >= p.vocab) return 0.f;
    return at * __builtin_amdgcn_exp2f((teacher_logit(p, r * k + j) - ref) * p.c);
  };
  // The entries that the teacher's tokens or the true one take from are written again, whole; a
  // token named twice by its first mention. Up to 64 of them lie one to a lane of the group's first
  // wave, or four to each of 16 lanes, which load them ahead of the dense pass (22.9 -> 20.7 us at
  // 32768 x 256; ahead of a workgroup's pass 107 -> 138 us at 2048 x 65536 bf16, all of which waits for them).
  constexpr int LANES = NT == 16 ? 16 : 64, E = 64 / LANES;
  const bool few = k <= 64, mine = few && G::tid() < LANES, truth = hard && tgt >= lo && tgt < hi;
  int eid[E];
  float ew[E], ex[E], tx = 0.f;
  const auto load_entries = [&] {
    if (!mine) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = e * LANES + G::tid();
      const int64_t id = j < k ? teacher_id(p, r * k + j) : -1;
      eid[e] = id >= lo && id < hi ? (int)id : -1;
      ew[e] = eid[e] >= 0 ? weight(id, j) : 0.f;
      ex[e] = eid[e] >= 0 ? (float)x[eid[e]] : 0.f;
    }
    if (truth) tx = (float)x[tgt];
  };
  if (NT == 16) load_entries();
  chunk_map<G>(x, dx, lo, hi, f);
  int* ids = sids[G::slot()];
  float* wt = sweight[G::slot()];
  if (NT == 16 || !few) {
    if (few) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        ids[e * LANES + G::tid()] = eid[e];
        wt[e * LANES + G::tid()] = ew[e];
      }
    } else {
      for (int j = G::tid(); j < k; j += G::NT) {
        const int64_t id = teacher_id(p, r * k + j);
        ids[j] = id >= lo && id < hi ? (int)id : -1;
        wt[j] = weight(id, j);
      }
    }
  }
  G::sync();
  if (few && !mine) return;   // only now: waves that are done make room for the next workgroup's
  if (NT > 16) load_entries();
  const auto whole = [&](int i, float xi, float take) {
    dx[i] = (T)(f(xi) - take - (hard && i == tgt ? b : 0.f));
  };
  const auto mentions = [&](int i, int j, float& take) {   // in LDS, of the j-th entry; first one?
    bool first = true;
    for (int l = 0; l < k; ++l) {
      const bool same = ids[l] == i;
      take += same ? wt[l] : 0.f;
      first = first && !(same && l < j);
    }
    return first;
  };
  bool named = false;   // the true token is among the entries, some thread knows
  if (few) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = e * LANES + G::tid();
      if (NT == 16 ? e * LANES >= k : !__ballot(eid[e] >= 0)) break;
      float take = 0.f;
      bool first = true;
      if constexpr (NT == 16) {
        if (eid[e] >= 0) first = mentions(eid[e], j, take);
      } else {
        for (int l = 0; l < k; ++l) {
          const bool same = __builtin_amdgcn_readlane(eid[0], l) == eid[0];
          const float wl = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ew[0]), l));
          take += same ? wl : 0.f;
          first = first && !(same && l < j);
        }
      }
      if (eid[e] >= 0 && first) whole(eid[e], ex[e], take);
      named = named || (truth && eid[e] == (int)tgt);
    }
    if (truth) {
      if constexpr (NT == 16) named = G::max(named ? 1.f : 0.f, nullptr) != 0.f;
      else named = __ballot(named) != 0;
      if (!named && G::tid() == 0) whole((int)tgt, tx, 0.f);
    }
    return;
  }
  for (int j = G::tid(); j < k; j += G::NT) {
    const int i = ids[j];
    if (i < 0) continue;
    float take = 0.f;
    if (mentions(i, j, take)) whole(i, (float)x[i], take);
  }
  if (G::tid() == 0 && truth) {
    for (int l = 0; l < k; ++l) named = named || ids[l] == tgt;
    if (!named) whole((int)tgt, (float)x[tgt], 0.f);
  }
}

// ---- host -----------------------------------------------------------------------------------
constexpr int64_t kRowGrid = 1 << 23;   // workgroups of a grid's first axis: 2^31 threads

template <typename A>
static int32_t check_rows(const A* a, const char* who) {
  M3S_REQUIRE(a != nullptr, "%s: args is NULL", who);
  M3S_REQUIRE(a->struct_size == (int32_t)sizeof(A), "%s: struct_size %d != %d (ABI mismatch)", who,
              a->struct_size, (int)sizeof(A));
  M3S_REQUIRE(a->dtype == M3S_DTYPE_BF16 || a->dtype == M3S_DTYPE_F32, "%s: bad dtype", who);
  M3S_REQUIRE(a->batch >= 0 && a->seqlen >= 0 && (int64_t)a->batch * a->seqlen < (1ll << 31),
              "%s: bad row count (%d x %d)", who, a->batch, a->seqlen);
  M3S_REQUIRE(a->vocab > 0 && a->vocab < (1 << 30), "%s: vocab %d must be in [1, 2^30)", who, a->vocab);
  // 1 / T, log2(e) / T and T^2 stay far from float32's ends
  M3S_REQUIRE(a->temperature >= 0.99e-6f && a->temperature <= 1.01e6f,
              "%s: temperature must be in [1e-6, 1e6]", who);
  return 0;
}
template <typename A>
static int32_t check_logits(const A* a, const char* who) {
  const uintptr_t es = a->dtype == M3S_DTYPE_BF16 ? 2 : 4;
  M3S_REQUIRE(a->logits.ptr && (uintptr_t)a->logits.ptr % es == 0, "%s: logits NULL or misaligned", who);
  M3S_REQUIRE(a->logits.stride_b >= 0 && a->logits.stride_t >= 0, "%s: negative logits stride", who);
  return 0;
}
// The threads to a row: `part` says that 16 lanes can do the call at all.
static int row_threads(int64_t rows, int vocab, bool part) {
  if (part && vocab <= kPartVocab && rows >= kPartRows) return 16;
  return vocab <= kWaveHeld || (vocab <= kWaveVocab && rows >= kWaveRows) ? 64 : 256;
}
// The backward's equal chunks of a row, at most kBwdPieces pieces to a thread, whole 16-byte pieces.
// A last chunk of what full ones leave would idle most of its threads: 16384 x 10000 in bf16, which is
// one full chunk and a fifth of one, took 189 us so and 145 as two equal ones (115 by now).
template <typename T, typename P>
static void set_chunks(P& p, int nt) {
  constexpr int N = Piece<T>::N;
  const int most = nt * kBwdPieces * N;
  p.chunks = (p.vocab + most - 1) / most;
  p.chunk = ((p.vocab + p.chunks - 1) / p.chunks + N - 1) / N * N;
}
// Rows from one stride_b to the next: all of them where the batch axis continues the other.
template <typename A>
static int row_period(const A* a) {
  const bool one = a->batch == 1 || a->logits.stride_b == (int64_t)a->seqlen * a->logits.stride_t;
  return one ? a->batch * a->seqlen : a->seqlen;
}
// Logits to a piece: whole 16-byte pieces.
static int row_share(int vocab, int split) { return ((vocab + split - 1) / split + 7) / 8 * 8; }
// Pieces to a row: where the rows alone leave most of the 256 CUs idle, enough for two workgroups
// to each, of at least kPieceMin logits; with alternatives the pieces' best together stay within
// what the joining workgroup ranks. 1: whole rows. 37 rows of 50001: distillation forward 17 us whole,
// 8 cut; one row of 131072 with 20 alternatives 10 us cut, in two launches of 3 to 6.
constexpr int kPieceMin = 4096, kSplitMax = 64;
static int row_split(int64_t rows, int vocab, int top) {
  int64_t split = std::min<int64_t>({512 / std::max<int64_t>(rows, 1), vocab / kPieceMin, kSplitMax});
  if (top) split = std::min<int64_t>(split, 1024 / top);
  if (split < 2) return 1;
  const int share = row_share(vocab, (int)split);
  return (vocab + share - 1) / share;
}

static LogprobParams logprob_params(const m3s_logprob_args* a) {
  LogprobParams p;
  p.logits = a->logits;
  p.targets = a->targets;
  p.logp = a->logp;
  p.entropy = a->entropy;
  p.stats = a->stats;
  p.top_logp = a->top_logp;
  p.top_ids = a->top_ids;
  p.dlogp = a->dlogp;
  p.dentropy = a->dentropy;
  p.dtop = a->dtop_logp;
  p.dlogits = a->dlogits;
  p.ignore = a->ignore_index;
  p.rows = (int64_t)a->batch * a->seqlen;
  p.seqlen = row_period(a);
  p.vocab = a->vocab;
  p.top = a->top;
  p.part = static_cast<float*>(a->workspace);
  p.inv_t = (float)(1.0 / a->temperature);
  p.c = (float)(1.4426950408889634 / a->temperature);
  return p;
}

static DistillParams distill_params(const m3s_distill_args* a) {
  DistillParams p;
  p.logits = a->logits;
  p.ids = a->teacher_ids;
  p.teacher = a->teacher_logits;
  p.targets = a->targets;
  p.kd = a->kd;
  p.nll = a->nll;
  p.stats = a->stats;
  p.dkd = a->dkd;
  p.dnll = a->dnll;
  p.dlogits = a->dlogits;
  p.ignore = a->ignore_index;
  p.rows = (int64_t)a->batch * a->seqlen;
  p.seqlen = row_period(a);
  p.vocab = a->vocab;
  p.k = a->teacher_k;
  p.part = static_cast<float*>(a->workspace);
  p.id_bytes = a->id_bytes;
  p.teacher_bf16 = a->teacher_dtype == M3S_DTYPE_BF16;
  p.temp = a->temperature;
  p.inv_t = (float)(1.0 / a->temperature);
  p.c = (float)(1.4426950408889634 / a->temperature);
  p.c1 = kLog2e;
  return p;
}

template <typename P>
static void launch_kernel(void (*f)(P), int64_t blocks, const P& p, hipStream_t s, int lds = 0) {
  const int64_t x = std::min(kRowGrid, blocks), y = (blocks + x - 1) / x;   // 2^39: more than memory holds
  hipLaunchKernelGGL(f, dim3((unsigned)x, (unsigned)y), dim3(kRowThreads), lds, s, p);
}
// The LDS for a backward of `own` bytes of its own: what leaves room for n workgroups on a CU (the
// middle of it) where rows of float32 take a workgroup a chunk and its threads four pieces. Eight fit,
// but then the loads and stores of so many chunks of 13 to 16 KB meet in HBM: the log-probabilities' at
// 8192 x 32000 and 8192 x 50001 take 338 and 521 us with four, 398 and 607 with five, 417 and 602 with
// eight. The distillation's workgroups last longer behind the dense pass, the more so with more teacher
// tokens: with 16 they take 341 and 525 with six, 345 and 578 with seven, 416 and 620 with eight, with 32
// 365 and 556, 355 and 543, 425 and 629, with 64 402 and 622, 377 and 578, 442 and 636. Smaller chunks
// want all eight (65536 x 5000: the distillation's 630 us with six, 488 with eight), and so do bf16's,
// half the bytes: 5 to 8% are won at some lengths (16384 x 32000) and lost at others (40000 x 10000).
constexpr int kLogprobGroups = 4;
static int distill_groups(int k) { return k <= 16 ? 6 : 7; }
template <typename G, typename T, typename P>
static int bwd_lds(const P& p, int n, int own) {
  const bool heavy = G::NT == 256 && sizeof(T) == 4 && p.chunk > 3 * G::NT * Piece<T>::N;
  return heavy ? 80 * 1024 / n + 80 * 1024 / (n + 1) - own : 0;
}
// f(group): the threads to a row
template <typename F>
static void with_group(int nt, F&& f) {
  if (nt == 16) f(Group<16>());
  else if (nt == 64) f(Group<64>());
  else f(Group<256>());
}
// Pieces of a thread's batch: 16 logits, or one piece where a wave holds the whole row so.
template <typename T>
constexpr int kBatch = 16 / Piece<T>::N;

template <bool TOP, typename T>
static void launch_logprob_fwd(const LogprobParams& p, hipStream_t s) {
  constexpr int U = kBatch<T>;
  if (p.split > 1) {
    launch_kernel(logprob_piece_kernel<TOP, U, T>, p.rows * p.split, p, s);
    launch_kernel(logprob_join_kernel<TOP, T>, p.rows, p, s);
    return;
  }
  int nt = row_threads(p.rows, p.vocab, !TOP || (p.top <= kPartTop && p.vocab <= kPartPick));
  if (TOP && p.vocab > kWaveHeld) nt = 256;   // a wave picks alternatives of a row that it holds
  with_group(nt, [&](auto g) {
    constexpr int NT = decltype(g)::NT, ROWS = decltype(g)::ROWS;
    const int64_t blocks = (p.rows + ROWS - 1) / ROWS;
    if constexpr (NT == 64) {
      if (p.vocab <= 64 * Piece<T>::N) return launch_kernel(logprob_fwd_kernel<TOP, NT, 1, T>, blocks, p, s);
    }
    launch_kernel(logprob_fwd_kernel<TOP, NT, U, T>, blocks, p, s);
  });
}
template <int MODE, typename T>
static void launch_distill_fwd(const DistillParams& p, hipStream_t s) {
  constexpr int U = kBatch<T>;
  if (p.split > 1) {
    launch_kernel(distill_piece_kernel<MODE, U, T>, p.rows * p.split, p, s);
    launch_kernel(distill_join_kernel<MODE, T>, p.rows, p, s);
    return;
  }
  with_group(row_threads(p.rows, p.vocab, p.k <= kPartTeacher), [&](auto g) {
    constexpr int NT = decltype(g)::NT, ROWS = decltype(g)::ROWS;
    launch_kernel(distill_fwd_kernel<MODE, NT, U, T>, (p.rows + ROWS - 1) / ROWS, p, s);
  });
}
template <typename T>
static void launch_logprob_bwd(LogprobParams& p, hipStream_t s) {
  const int nt = row_threads(p.rows, p.vocab, true);
  set_chunks<T>(p, nt);
  with_group(nt, [&](auto g) {
    constexpr int NT = decltype(g)::NT, ROWS = decltype(g)::ROWS;
    const int lds = bwd_lds<decltype(g), T>(p, kLogprobGroups, 8 * (kTopMax + 1));
    launch_kernel(logprob_bwd_kernel<NT, T>, (p.rows * p.chunks + ROWS - 1) / ROWS, p, s, lds);
  });
}
template <bool DUAL, typename T>
static void launch_distill_bwd(DistillParams& p, hipStream_t s) {
  const int nt = row_threads(p.rows, p.vocab, p.k <= kPartTeacher);
  set_chunks<T>(p, nt);
  with_group(nt, [&](auto g) {
    constexpr int NT = decltype(g)::NT, ROWS = decltype(g)::ROWS;
    const int lds = bwd_lds<decltype(g), T>(p, distill_groups(p.k), 8 * (kTeacherMax + 1));
    launch_kernel(distill_bwd_kernel<DUAL, NT, T>, (p.rows * p.chunks + ROWS - 1) / ROWS, p, s, lds);
  });
}

static int64_t logprob_scratch(int64_t rows, int vocab, int top) {
  const int split = row_split(rows, vocab, top);
  return split == 1 ? 0 : rows * split * (3 + 2 * top) * 4;
}
static int64_t distill_scratch(int64_t rows, int vocab) {
  const int split = row_split(rows, vocab, 0);
  return split == 1 ? 0 : rows * split * 3 * 4;
}
// Rows are cut where the call brings the scratch for it, and stay whole (the same results to
// rounding, later) where it does not.
template <typename P>
static void set_split(P& p, int64_t need, int64_t given, int top) {
  p.split = need > 0 && p.part && given >= need ? row_split(p.rows, p.vocab, top) : 1;
  p.share = row_share(p.vocab, p.split);
}
template <typename A>
static int32_t check_scratch(const A* a, const char* who) {
  M3S_REQUIRE(a->workspace_bytes >= 0 && (uintptr_t)a->workspace % 16 == 0,
              "%s: workspace must be 16-byte aligned", who);
  return 0;
}

}  // namespace m3s

using namespace m3s;

extern "C" int64_t m3s_logprob_workspace_bytes(int64_t rows, int32_t vocab, int32_t top) {
  if (rows < 0 || rows >= (1ll << 31) || vocab <= 0 || vocab >= (1 << 30) || top < 0 || top > kTopMax) return -1;
  return logprob_scratch(rows, vocab, top);
}

extern "C" int64_t m3s_distill_workspace_bytes(int64_t rows, int32_t vocab) {
  if (rows < 0 || rows >= (1ll << 31) || vocab <= 0 || vocab >= (1 << 30)) return -1;
  return distill_scratch(rows, vocab);
}

extern "C" int32_t m3s_logprob_fwd(const m3s_logprob_args* a, void* stream) {
  clear_error();
  if (int32_t rc = check_rows(a, "m3s_logprob_fwd")) return rc;
  M3S_REQUIRE(a->top >= 0 && a->top <= kTopMax && a->top <= a->vocab,
              "m3s_logprob_fwd: top %d must be in [0, %d] and at most the vocabulary", a->top, kTopMax);
  if (a->batch == 0 || a->seqlen == 0) return 0;
  if (int32_t rc = check_logits(a, "m3s_logprob_fwd")) return rc;
  M3S_REQUIRE(a->entropy && (!a->targets || a->logp) && (!a->top || (a->top_logp && a->top_ids)),
              "m3s_logprob_fwd: NULL pointer");
  if (int32_t rc = check_scratch(a, "m3s_logprob_fwd")) return rc;
  LogprobParams p = logprob_params(a);
  set_split(p, logprob_scratch(p.rows, p.vocab, p.top), a->workspace_bytes, p.top);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool b = a->dtype == M3S_DTYPE_BF16;
  if (p.top) b ? launch_logprob_fwd<true, bf16>(p, s) : launch_logprob_fwd<true, float>(p, s);
  else b ? launch_logprob_fwd<false, bf16>(p, s) : launch_logprob_fwd<false, float>(p, s);
  return launch_status("m3s_logprob_fwd");
}

extern "C" int32_t m3s_logprob_bwd(const m3s_logprob_args* a, void* stream) {
  clear_error();
  if (int32_t rc = check_rows(a, "m3s_logprob_bwd")) return rc;
  M3S_REQUIRE(a->top >= 0 && a->top <= kTopMax && a->top <= a->vocab,
              "m3s_logprob_bwd: top %d must be in [0, %d] and at most the vocabulary", a->top, kTopMax);
  if (a->batch == 0 || a->seqlen == 0) return 0;
  if (int32_t rc = check_logits(a, "m3s_logprob_bwd")) return rc;
  const uintptr_t es = a->dtype == M3S_DTYPE_BF16 ? 2 : 4;
  M3S_REQUIRE(a->stats && a->dlogits && (uintptr_t)a->dlogits % es == 0 && (!a->dlogp || a->targets) &&
                  (!a->dtop_logp || !a->top || a->top_ids),
              "m3s_logprob_bwd: NULL or misaligned pointer");
  LogprobParams p = logprob_params(a);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == M3S_DTYPE_BF16) launch_logprob_bwd<bf16>(p, s);
  else launch_logprob_bwd<float>(p, s);
  return launch_status("m3s_logprob_bwd");
}

static int32_t check_distill(const m3s_distill_args* a, const char* who) {
  if (int32_t rc = check_rows(a, who)) return rc;
  M3S_REQUIRE(a->teacher_k >= 1 && a->teacher_k <= kTeacherMax, "%s: teacher_k %d must be in [1, %d]", who,
              a->teacher_k, kTeacherMax);
  M3S_REQUIRE(a->id_bytes == 4 || a->id_bytes == 8, "%s: ids of %d bytes, must be 4 or 8", who, a->id_bytes);
  M3S_REQUIRE(a->teacher_dtype == M3S_DTYPE_BF16 || a->teacher_dtype == M3S_DTYPE_F32, "%s: bad teacher dtype",
              who);
  if (a->batch == 0 || a->seqlen == 0) return 0;
  if (int32_t rc = check_logits(a, who)) return rc;
  M3S_REQUIRE(a->teacher_ids && a->teacher_logits, "%s: NULL pointer", who);
  return 0;
}

extern "C" int32_t m3s_distill_fwd(const m3s_distill_args* a, void* stream) {
  clear_error();
  if (int32_t rc = check_distill(a, "m3s_distill_fwd")) return rc;
  if (a->batch == 0 || a->seqlen == 0) return 0;
  M3S_REQUIRE(a->kd && (a->targets == nullptr) == (a->nll == nullptr), "m3s_distill_fwd: NULL pointer");
  if (int32_t rc = check_scratch(a, "m3s_distill_fwd")) return rc;
  DistillParams p = distill_params(a);
  set_split(p, distill_scratch(p.rows, p.vocab), a->workspace_bytes, 0);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool b = a->dtype == M3S_DTYPE_BF16, dual = p.targets && p.temp != 1.f;
  if (dual) b ? launch_distill_fwd<kDual, bf16>(p, s) : launch_distill_fwd<kDual, float>(p, s);
  else b ? launch_distill_fwd<kSingle, bf16>(p, s) : launch_distill_fwd<kSingle, float>(p, s);
  return launch_status("m3s_distill_fwd");
}

extern "C" int32_t m3s_distill_bwd(const m3s_distill_args* a, void* stream) {
  clear_error();
  if (int32_t rc = check_distill(a, "m3s_distill_bwd")) return rc;
  if (a->batch == 0 || a->seqlen == 0) return 0;
  const uintptr_t es = a->dtype == M3S_DTYPE_BF16 ? 2 : 4;
  M3S_REQUIRE(a->stats && a->dlogits && (uintptr_t)a->dlogits % es == 0 && (!a->dnll || a->targets),
              "m3s_distill_bwd: NULL or misaligned pointer");
  DistillParams p = distill_params(a);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool b = a->dtype == M3S_DTYPE_BF16, dual = p.dkd && p.dnll && p.temp != 1.f;
  if (dual) b ? launch_distill_bwd<true, bf16>(p, s) : launch_distill_bwd<true, float>(p, s);
  else b ? launch_distill_bwd<false, bf16>(p, s) : launch_distill_bwd<false, float>(p, s);
  return launch_status("m3s_distill_bwd");
}
