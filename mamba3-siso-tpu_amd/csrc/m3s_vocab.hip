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
#include <algorithm>

#include "m3s_common.h"
#include "m3s_internal.h"

namespace m3s {

constexpr int kRowThreads = 256;
constexpr int kTopMax = 64;        // alternatives of a row
constexpr int kTeacherMax = 256;   // teacher tokens of a row: one a thread
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

// ---- reductions over a workgroup of four waves ----------------------------------------------
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
// Each returns the same value to every thread; `tmp` holds four floats and is free afterwards.
__device__ __forceinline__ float block_max(float v, float* tmp) {
  v = wave_max(v);
  if (lane_id() == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  v = fmaxf(fmaxf(tmp[0], tmp[1]), fmaxf(tmp[2], tmp[3]));
  __syncthreads();
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* tmp) {
  v = wave_total(v);
  if (lane_id() == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (tmp[0] + tmp[1]) + (tmp[2] + tmp[3]);
  __syncthreads();
  return v;
}

// ---- running sums of a row ------------------------------------------------------------------
// s = sum 2^{c (x - m)}, t = sum of the same times (x - m), s1 = sum 2^{c1 (x - m)}. A row of -inf
// keeps m = -inf and zeros; a NaN or +inf makes the sums NaN (fmaxf drops the NaN, s does not).
enum { kPlain = 0, kEntropy = 1, kDual = 2 };
template <int MODE>
struct RowSums {
  float m = kNegInf, s = 0.f, t = 0.f, s1 = 0.f;

  // m grows to at least `to`; the sums follow
  __device__ __forceinline__ void raise(float to, float c, float c1) {
    const float mn = fmaxf(m, to);
    const float ref = mn == kNegInf ? 0.f : mn;
    const float gap = fmaxf(m - ref, -1e30f);   // 0 * -1e30, not 0 * -inf, while s = 0
    const float f = __builtin_amdgcn_exp2f(gap * c);
    if constexpr (MODE == kEntropy) t = (t + s * gap) * f;
    s *= f;
    if constexpr (MODE == kDual) s1 *= __builtin_amdgcn_exp2f(gap * c1);
    m = mn;
  }
  template <int N>
  __device__ __forceinline__ void add(const float* x, float c, float c1) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    raise(top, c, c1);
    const float ref = m == kNegInf ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = x[i] - ref;
      const float e = __builtin_amdgcn_exp2f(d * c);
      s += e;
      if constexpr (MODE == kEntropy) t += e * fmaxf(d, -1e30f);
      if constexpr (MODE == kDual) s1 += __builtin_amdgcn_exp2f(d * c1);
    }
  }
  __device__ __forceinline__ void join_block(float c, float c1, float* tmp) {
    raise(block_max(m, tmp), c, c1);
    s = block_sum(s, tmp);
    if constexpr (MODE == kEntropy) t = block_sum(t, tmp);
    if constexpr (MODE == kDual) s1 = block_sum(s1, tmp);
  }
};

// One pass over n logits by the workgroup.
template <int MODE, typename T>
__device__ __forceinline__ void row_pass(RowSums<MODE>& r, const T* __restrict__ x, int n, float c,
                                         float c1) {
  constexpr int N = Piece<T>::N, U = 16 / N, HOP = kRowThreads * U;
  const int full = n / N, tail = n - full * N, tid = threadIdx.x;
  for (int p = 0; p < full; p += HOP) {
    float v[U * N];
    if (p + HOP <= full) {
#pragma unroll
      for (int u = 0; u < U; ++u) Piece<T>::load(x + (int64_t)(p + u * kRowThreads + tid) * N, v + u * N);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = p + u * kRowThreads + tid;
        if (at < full) {
          Piece<T>::load(x + (int64_t)at * N, v + u * N);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) v[u * N + i] = kNegInf;
        }
      }
    }
    r.template add<U * N>(v, c, c1);
  }
  if (tid < tail) {
    const float v = (float)x[(int64_t)full * N + tid];
    r.template add<1>(&v, c, c1);
  }
}

template <typename T>
__device__ __forceinline__ const T* row_at(const m3s_blx& b, int64_t r, int seqlen) {
  const int64_t i = r / seqlen;
  return static_cast<const T*>(b.ptr) + i * b.stride_b + (r - i * seqlen) * b.stride_t;
}

// The k best of a row, one round of (largest value, lowest index) each. For rows without NaN.
template <typename T, typename OUT>
__device__ __forceinline__ void pick_rounds(const T* __restrict__ x, int n, int k, float* tmp,
                                            int* itmp, OUT&& out) {
  float last = __builtin_inff();
  int last_i = -1;
  for (int j = 0; j < k; ++j) {
    float best = kNegInf;
    int best_i = 0x7fffffff;
    for (int i = threadIdx.x; i < n; i += kRowThreads) {
      const float v = (float)x[i];
      const bool left = v < last || (v == last && i > last_i);
      if (left && (v > best || (v == best && i < best_i))) {
        best = v;
        best_i = i;
      }
    }
    const float v = block_max(best, tmp);
    int i = best == v ? best_i : 0x7fffffff;
#pragma unroll
    for (int o = 32; o; o >>= 1) i = min(i, __shfl_xor(i, o));
    if (lane_id() == 0) itmp[threadIdx.x >> 6] = i;
    __syncthreads();
    i = min(min(itmp[0], itmp[1]), min(itmp[2], itmp[3]));
    __syncthreads();
    if (threadIdx.x == 0) out(j, v, i);
    last = v;
    last_i = i;
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
  int64_t ignore, rows;
  int seqlen, vocab, top, chunks;
  float temp, inv_t, c;
};

template <typename T>
__global__ void __launch_bounds__(kRowThreads) logprob_fwd_kernel(const LogprobParams p) {
  __shared__ float tmp[4];
  __shared__ int itmp[4];
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const int64_t tgt = p.targets ? p.targets[r] : 0;
    if (p.targets && tgt == p.ignore) {   // no token here: the logits are not read
      if (threadIdx.x == 0) {
        p.logp[r] = p.entropy[r] = 0.f;
        p.stats[3 * r] = p.stats[3 * r + 1] = p.stats[3 * r + 2] = 0.f;
      }
      for (int j = threadIdx.x; j < p.top; j += kRowThreads) {
        p.top_logp[r * p.top + j] = kNegInf;
        p.top_ids[r * p.top + j] = -1;
      }
      continue;
    }
    const T* x = row_at<T>(p.logits, r, p.seqlen);
    RowSums<kEntropy> sum;
    row_pass<kEntropy>(sum, x, p.vocab, p.c, 0.f);
    sum.join_block(p.c, 0.f, tmp);
    const bool empty = sum.m == kNegInf && sum.s == 0.f;
    const float logs = logf(sum.s);
    const auto logp = [&](float v) { return empty ? kNegInf : (v - sum.m) / p.temp - logs; };
    if (threadIdx.x == 0) {
      const float h = empty ? 0.f : logs - sum.t / (p.temp * sum.s);
      p.entropy[r] = h;
      p.stats[3 * r] = sum.m;
      p.stats[3 * r + 1] = sum.s;
      p.stats[3 * r + 2] = h;
      if (p.targets) p.logp[r] = tgt >= 0 && tgt < p.vocab ? logp((float)x[tgt]) : __builtin_nanf("");
    }
    if (p.top == 0) continue;
    if (sum.s != sum.s) {   // NaN or +inf among the logits: no order to report
      for (int j = threadIdx.x; j < p.top; j += kRowThreads) {
        p.top_logp[r * p.top + j] = __builtin_nanf("");
        p.top_ids[r * p.top + j] = -1;
      }
      continue;
    }
    pick_rounds(x, p.vocab, p.top, tmp, itmp, [&](int j, float v, int i) {
      p.top_logp[r * p.top + j] = logp(v);
      p.top_ids[r * p.top + j] = i;
    });
  }
}

// The dense part of a gradient: f(d) for every logit of a chunk (blockIdx.x = row * chunks + chunk),
// d = x - m. Returns nothing to the caller but the chunk's bounds.
constexpr int kBwdPieces = 4;
template <typename T, typename F>
__device__ __forceinline__ void chunk_map(const T* __restrict__ x, T* __restrict__ dx, int lo, int hi,
                                          F&& f) {
  constexpr int N = Piece<T>::N;
  const int n = hi - lo, full = n / N, tid = threadIdx.x;
  float v[kBwdPieces * N];
#pragma unroll
  for (int u = 0; u < kBwdPieces; ++u) {
    const int at = u * kRowThreads + tid;
    if (at < full) Piece<T>::load(x + lo + at * N, v + u * N);
  }
#pragma unroll
  for (int u = 0; u < kBwdPieces; ++u) {
    const int at = u * kRowThreads + tid;
    if (at < full) {
      float o[N];
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = f(v[u * N + i]);
      Piece<T>::store(dx + lo + at * N, o);
    }
  }
  const int at = full * N + tid;
  if (at < n) dx[lo + at] = (T)f((float)x[lo + at]);
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) logprob_bwd_kernel(const LogprobParams p) {
  constexpr int CHUNK = kRowThreads * kBwdPieces * Piece<T>::N;
  __shared__ int ids[kTopMax];
  __shared__ float gtop[kTopMax];
  for (int64_t w = blockIdx.x; w < p.rows * p.chunks; w += gridDim.x) {
    const int64_t r = w / p.chunks;
    const int lo = (int)(w - r * p.chunks) * CHUNK, hi = min(lo + CHUNK, p.vocab);
    const T* x = row_at<T>(p.logits, r, p.seqlen);
    T* dx = static_cast<T*>(p.dlogits) + r * p.vocab;
    const int64_t tgt = p.targets ? p.targets[r] : -1;
    const float m = p.stats[3 * r], s = p.stats[3 * r + 1], h = p.stats[3 * r + 2];
    // an ignored row, and one of nothing but -inf, has s = 0 and no gradient
    if (s == 0.f) {
      for (int i = lo + threadIdx.x; i < hi; i += kRowThreads) dx[i] = (T)0.f;
      continue;
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
    chunk_map(x, dx, lo, hi, f);
    // then the entries that a token or an alternative adds to, whole
    for (int j = threadIdx.x; j < top; j += kRowThreads) {
      ids[j] = (int)p.top_ids[r * top + j];
      gtop[j] = p.dtop[r * top + j] * p.inv_t;
    }
    __syncthreads();
    for (int j = threadIdx.x; j < top; j += kRowThreads) {
      const int i = ids[j];
      if (i >= lo && i < hi) dx[i] = (T)(f((float)x[i]) + gtop[j] + (i == tgt ? gl : 0.f));
    }
    if (threadIdx.x == 0 && p.dlogp && tgt >= lo && tgt < hi) {
      bool alone = true;
      for (int j = 0; j < top; ++j) alone = alone && ids[j] != tgt;
      if (alone) dx[tgt] = (T)(f((float)x[tgt]) + gl);
    }
    __syncthreads();
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
  int64_t ignore, rows;
  int seqlen, vocab, k, chunks, id_bytes, teacher_bf16;
  float temp, inv_t, c, c1;
};

__device__ __forceinline__ int64_t teacher_id(const DistillParams& p, int64_t at) {
  return p.id_bytes == 8 ? static_cast<const int64_t*>(p.ids)[at] : (int64_t)static_cast<const int32_t*>(p.ids)[at];
}
__device__ __forceinline__ float teacher_logit(const DistillParams& p, int64_t at) {
  return p.teacher_bf16 ? (float)static_cast<const bf16*>(p.teacher)[at] : static_cast<const float*>(p.teacher)[at];
}

// stats (rows, 5): m, sum e^{d / T}, sum e^d, the teacher's maximum and its sum (0: no entry; NaN: an
// id outside the vocabulary, or a NaN).
template <typename T>
__global__ void __launch_bounds__(kRowThreads) distill_fwd_kernel(const DistillParams p) {
  __shared__ float tmp[4];
  const int tid = threadIdx.x;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = row_at<T>(p.logits, r, p.seqlen);
    float u = kNegInf;
    int64_t id = -1;
    if (tid < p.k) {
      id = teacher_id(p, r * p.k + tid);
      if (id >= 0) u = teacher_logit(p, r * p.k + tid);
      if (id >= p.vocab) u = __builtin_nanf("");
    }
    const float tm = block_max(u, tmp);
    const float ref = tm == kNegInf ? 0.f : tm;
    const float e = __builtin_amdgcn_exp2f((u - ref) * p.c);
    const float ts = block_sum(e, tmp);
    const int64_t tgt = p.targets ? p.targets[r] : 0;
    const bool soft = ts != 0.f, hard = p.targets && tgt != p.ignore;
    float* stats = p.stats + 5 * r;
    if (!soft && !hard) {   // nothing to learn here: the logits are not read
      if (tid == 0) {
        p.kd[r] = 0.f;
        if (p.nll) p.nll[r] = 0.f;
        stats[0] = stats[1] = stats[2] = stats[3] = stats[4] = 0.f;
      }
      continue;
    }
    RowSums<kDual> sum;
    row_pass<kDual>(sum, x, p.vocab, p.c, p.c1);
    sum.join_block(p.c, p.c1, tmp);
    const bool empty = sum.m == kNegInf && sum.s == 0.f;
    float term = 0.f;
    if (e != 0.f) {   // w (log w - log q)
      const float w = e / ts;
      const float lw = (u - ref) / p.temp - logf(ts);
      const float xi = id >= 0 && id < p.vocab ? (float)x[id] : __builtin_nanf("");
      const float lq = empty ? kNegInf : (xi - sum.m) / p.temp - logf(sum.s);
      term = w * (lw - lq);
    }
    const float kd = block_sum(term, tmp);
    if (tid == 0) {
      p.kd[r] = soft ? p.temp * p.temp * kd : 0.f;
      stats[0] = sum.m;
      stats[1] = sum.s;
      stats[2] = sum.s1;
      stats[3] = ref;
      stats[4] = ts;
      if (p.nll) {
        float v = 0.f;
        if (hard) {
          v = tgt < 0 || tgt >= p.vocab ? __builtin_nanf("")
              : empty                   ? __builtin_inff()
                                        : logf(sum.s1) - ((float)x[tgt] - sum.m);
        }
        p.nll[r] = v;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) distill_bwd_kernel(const DistillParams p) {
  constexpr int CHUNK = kRowThreads * kBwdPieces * Piece<T>::N;
  __shared__ int ids[kTeacherMax];
  __shared__ float wt[kTeacherMax];
  const int tid = threadIdx.x;
  for (int64_t w = blockIdx.x; w < p.rows * p.chunks; w += gridDim.x) {
    const int64_t r = w / p.chunks;
    const int lo = (int)(w - r * p.chunks) * CHUNK, hi = min(lo + CHUNK, p.vocab);
    const T* x = row_at<T>(p.logits, r, p.seqlen);
    T* dx = static_cast<T*>(p.dlogits) + r * p.vocab;
    const float* stats = p.stats + 5 * r;
    const float m = stats[0], s = stats[1], s1 = stats[2], ref = stats[3], ts = stats[4];
    const int64_t tgt = p.targets ? p.targets[r] : p.ignore;
    const bool soft = p.dkd && ts != 0.f, hard = p.dnll && tgt != p.ignore;
    if (s == 0.f || (!soft && !hard)) {   // no loss, or no distribution
      for (int i = lo + tid; i < hi; i += kRowThreads) dx[i] = (T)0.f;
      continue;
    }
    const float a = soft ? p.dkd[r] * p.temp : 0.f, as = ts != ts ? ts : a / s;
    float b = hard ? p.dnll[r] : 0.f;
    if (hard && (tgt < 0 || tgt >= p.vocab)) b = __builtin_nanf("");
    const float bs = b / s1;
    const auto f = [&](float v) {
      const float d = v - m;
      float o = 0.f;
      if (soft) o = as * __builtin_amdgcn_exp2f(d * p.c);
      if (hard) o += bs * __builtin_amdgcn_exp2f(d * p.c1);
      return o;
    };
    chunk_map(x, dx, lo, hi, f);
    const int k = soft ? p.k : 0;
    if (tid < k) {
      const int64_t id = teacher_id(p, r * k + tid);
      const bool there = id >= 0 && id < p.vocab;
      ids[tid] = there ? (int)id : -1;
      wt[tid] = there ? a * __builtin_amdgcn_exp2f((teacher_logit(p, r * k + tid) - ref) * p.c) / ts : 0.f;
    }
    __syncthreads();
    // entries that the teacher's tokens or the true one take from, whole: a token named twice
    // is written by its first mention
    if (tid < k && ids[tid] >= lo && ids[tid] < hi) {
      const int i = ids[tid];
      bool first = true;
      float take = 0.f;
      for (int j = 0; j < k; ++j) {
        if (ids[j] == i) {
          first = first && j >= tid;
          take += wt[j];
        }
      }
      if (first) dx[i] = (T)(f((float)x[i]) - take - (hard && i == tgt ? b : 0.f));
    }
    if (tid == 0 && hard && tgt >= lo && tgt < hi) {
      bool alone = true;
      for (int j = 0; j < k; ++j) alone = alone && ids[j] != tgt;
      if (alone) dx[tgt] = (T)(f((float)x[tgt]) - b);
    }
    __syncthreads();
  }
}

// ---- host -----------------------------------------------------------------------------------
constexpr int64_t kRowGrid = 1 << 20;

template <typename A>
static int32_t check_rows(const A* a, const char* who) {
  M3S_REQUIRE(a != nullptr, "%s: args is NULL", who);
  M3S_REQUIRE(a->struct_size == (int32_t)sizeof(A), "%s: struct_size %d != %d (ABI mismatch)", who,
              a->struct_size, (int)sizeof(A));
  M3S_REQUIRE(a->dtype == M3S_DTYPE_BF16 || a->dtype == M3S_DTYPE_F32, "%s: bad dtype", who);
  M3S_REQUIRE(a->batch >= 0 && a->seqlen >= 0 && (int64_t)a->batch * a->seqlen < (1ll << 31),
              "%s: bad row count (%d x %d)", who, a->batch, a->seqlen);
  M3S_REQUIRE(a->vocab > 0 && a->vocab < (1 << 30), "%s: vocab %d must be in [1, 2^30)", who, a->vocab);
  M3S_REQUIRE(a->temperature > 0.f && a->temperature <= 3.4e38f && 1.f / a->temperature <= 3.4e38f,
              "%s: temperature must be positive and finite", who);
  return 0;
}
template <typename A>
static int32_t check_logits(const A* a, const char* who) {
  const uintptr_t es = a->dtype == M3S_DTYPE_BF16 ? 2 : 4;
  M3S_REQUIRE(a->logits.ptr && (uintptr_t)a->logits.ptr % es == 0, "%s: logits NULL or misaligned", who);
  M3S_REQUIRE(a->logits.stride_b >= 0 && a->logits.stride_t >= 0, "%s: negative logits stride", who);
  return 0;
}
static int vocab_chunks(int vocab, int dtype) {
  const int chunk = kRowThreads * kBwdPieces * (dtype == M3S_DTYPE_BF16 ? 8 : 4);
  return (vocab + chunk - 1) / chunk;
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
  p.seqlen = a->seqlen;
  p.vocab = a->vocab;
  p.top = a->top;
  p.chunks = vocab_chunks(a->vocab, a->dtype);
  p.temp = a->temperature;
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
  p.seqlen = a->seqlen;
  p.vocab = a->vocab;
  p.k = a->teacher_k;
  p.chunks = vocab_chunks(a->vocab, a->dtype);
  p.id_bytes = a->id_bytes;
  p.teacher_bf16 = a->teacher_dtype == M3S_DTYPE_BF16;
  p.temp = a->temperature;
  p.inv_t = (float)(1.0 / a->temperature);
  p.c = (float)(1.4426950408889634 / a->temperature);
  p.c1 = kLog2e;
  return p;
}

template <typename P>
static void launch_rows(void (*fb)(P), void (*ff)(P), const P& p, int dtype, int64_t blocks, hipStream_t s) {
  const dim3 grid((unsigned)std::min(kRowGrid, blocks));
  if (dtype == M3S_DTYPE_BF16) hipLaunchKernelGGL(fb, grid, dim3(kRowThreads), 0, s, p);
  else hipLaunchKernelGGL(ff, grid, dim3(kRowThreads), 0, s, p);
}

}  // namespace m3s

using namespace m3s;

extern "C" int32_t m3s_logprob_fwd(const m3s_logprob_args* a, void* stream) {
  clear_error();
  if (int32_t rc = check_rows(a, "m3s_logprob_fwd")) return rc;
  M3S_REQUIRE(a->top >= 0 && a->top <= kTopMax && a->top <= a->vocab,
              "m3s_logprob_fwd: top %d must be in [0, %d] and at most the vocabulary", a->top, kTopMax);
  if (a->batch == 0 || a->seqlen == 0) return 0;
  if (int32_t rc = check_logits(a, "m3s_logprob_fwd")) return rc;
  M3S_REQUIRE(a->entropy && a->stats && (!a->targets || a->logp) && (!a->top || (a->top_logp && a->top_ids)),
              "m3s_logprob_fwd: NULL pointer");
  const LogprobParams p = logprob_params(a);
  launch_rows(logprob_fwd_kernel<bf16>, logprob_fwd_kernel<float>, p, a->dtype, p.rows,
              static_cast<hipStream_t>(stream));
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
  const LogprobParams p = logprob_params(a);
  launch_rows(logprob_bwd_kernel<bf16>, logprob_bwd_kernel<float>, p, a->dtype, p.rows * p.chunks,
              static_cast<hipStream_t>(stream));
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
  M3S_REQUIRE(a->teacher_ids && a->teacher_logits && a->stats, "%s: NULL pointer", who);
  return 0;
}

extern "C" int32_t m3s_distill_fwd(const m3s_distill_args* a, void* stream) {
  clear_error();
  if (int32_t rc = check_distill(a, "m3s_distill_fwd")) return rc;
  if (a->batch == 0 || a->seqlen == 0) return 0;
  M3S_REQUIRE(a->kd && (a->targets == nullptr) == (a->nll == nullptr), "m3s_distill_fwd: NULL pointer");
  const DistillParams p = distill_params(a);
  launch_rows(distill_fwd_kernel<bf16>, distill_fwd_kernel<float>, p, a->dtype, p.rows,
              static_cast<hipStream_t>(stream));
  return launch_status("m3s_distill_fwd");
}

extern "C" int32_t m3s_distill_bwd(const m3s_distill_args* a, void* stream) {
  clear_error();
  if (int32_t rc = check_distill(a, "m3s_distill_bwd")) return rc;
  if (a->batch == 0 || a->seqlen == 0) return 0;
  const uintptr_t es = a->dtype == M3S_DTYPE_BF16 ? 2 : 4;
  M3S_REQUIRE(a->dlogits && (uintptr_t)a->dlogits % es == 0 && (!a->dnll || a->targets),
              "m3s_distill_bwd: NULL or misaligned pointer");
  const DistillParams p = distill_params(a);
  launch_rows(distill_bwd_kernel<bf16>, distill_bwd_kernel<float>, p, a->dtype, p.rows * p.chunks,
              static_cast<hipStream_t>(stream));
  return launch_status("m3s_distill_bwd");
}
