// The language model's embedding on gfx950: the scaled lookup and the table's gradient.
//
//   forward:   y[t] = scale table[id_t]
//   backward:  dtable[v] = scale sum_{t : id_t = v} dy[t], v != padding_idx
//
// The lookup is a gather of whole rows, bound by HBM (the output; a byte LM's table stays in L2).
//
// The gradient is a sum of rows by token id. Adding rows into the table with atomics would make
// the result depend on the order of arrival and would serialise on the commonest ids (the first
// of 256 Zipf-distributed bytes stands on a sixth of all positions). So the positions are sorted
// by id, stably, and each id's rows stand together in position order:
//
//   1. least-significant-digit radix sort of (id, position), at most 9 bits a pass: one pass for
//      bytes, two for fewer than 2^18 ids. Ranks within a wave come from ballots (lanes with the same digit
//      find each other bit by bit), across waves and workgroups from digit counts, so the order
//      is that of the positions whatever runs first. Up to 4096 tokens one workgroup sorts in LDS.
//      The sort waits more than it works and fills few CUs: workgroups beside it clear the table.
//   2. run_sum: a wave adds a piece of 8 to 32 sorted rows, 256 columns of them. A run of equal
//      ids inside the piece is finished and written; one that crosses a border leaves a float32
//      partial sum.
//   3. finish: the workgroup of the piece that a crossing run starts in adds its partials, in order.
//
// Up to 1024 tokens a single launch does without the sort: each workgroup lists its own rows' tokens.
//
// Every sum is float32 in a fixed order, rounded once. The gradient reads dy once and writes the
// table once (a row that occurs twice): bound by HBM from a few MB on, by the launches below that.
//
// Measured: 32768 byte tokens (Zipf), D 768, float32: lookup 17.9 us (5.6 TB/s of output), gradient
// 34 us, of which run_sum 19 (5.3 TB/s of dy), the sort 9 and finish 6. 16384 tokens of 50001, D 1024:
// gradient 66 us, of which clearing 205 MB beside the four sort launches takes 38 (5.4 TB/s) and
// run_sum 25; cleared by a pass of its own behind the sort it took 96 in all. 777 tokens of
// 32003, D 515, bf16: 13.2 us in one launch (2.5 TB/s, the table's 33 MB), 16.4 sorted.
#include <algorithm>

#include "m3s_common.h"
#include "m3s_internal.h"

namespace m3s {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kDigits = 512;          // counters of a pass: digits of up to 9 bits
constexpr int kDigitBits = 9;
constexpr int kSortOne = 4096;        // tokens that one workgroup sorts alone, in LDS
constexpr int kSortRounds = kSortOne / kSortThreads;
constexpr int kSortBlocks = 64;       // workgroups of a larger sort, at most
// Waves of run_sum that make its pieces longer: longer pieces leave fewer partials, shorter ones more
// waves. The whole gradient at 32768 x 768 in pieces of 32 rows took 39 us, 45 and 56 with pieces of
// 16 and 8; at 16384 x 1024 (2048 waves) 65 against 68 and 78.
constexpr int64_t kRunWaves = 2048;

// W columns of a row, at any element alignment (gfx950 takes wide accesses there): 8 or 4 of bf16, 4
// of float32, or one of a row narrower than that. Lanes take W columns each and the last one steps back to the
// row's end: it and its neighbour then hold some columns both, read, add and write the same numbers
// for them, and no row needs a ragged edge.
template <int W> struct Cols { typedef float type __attribute__((ext_vector_type(W))); };
template <int W> using cols = typename Cols<W>::type;
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef bf16x8 bf16x8_u __attribute__((aligned(2)));
typedef bf16x4 bf16x4_u __attribute__((aligned(2)));
template <int W> struct Halves { typedef bf16x8_u type; };
template <> struct Halves<4> { typedef bf16x4_u type; };
template <typename T> constexpr int kCols = 16 / sizeof(T);

template <int W, typename T>
__device__ __forceinline__ cols<W> ld_cols(const T* p) {
  cols<W> v;
  if constexpr (W == 1) {
    v[0] = (float)p[0];
  } else if constexpr (sizeof(T) == 2) {
    const typename Halves<W>::type r = *reinterpret_cast<const typename Halves<W>::type*>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = (float)r[i];
  } else {
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      const f32x4 r = *reinterpret_cast<const f32x4_u*>(p + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j + i] = r[i];
    }
  }
  return v;
}
template <int W, typename T>
__device__ __forceinline__ void st_cols(T* p, cols<W> v) {
  if constexpr (W == 1) {
    p[0] = (T)v[0];
  } else if constexpr (sizeof(T) == 2) {
    typename Halves<W>::type r;
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] = (bf16)v[i];
    *reinterpret_cast<typename Halves<W>::type*>(p) = r;
  } else {
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      *reinterpret_cast<f32x4_u*>(p + j) = f32x4{v[j], v[j + 1], v[j + 2], v[j + 3]};
    }
  }
}

// ---- lookup -----------------------------------------------------------------------------
// Two forms, by measurement (us; in brackets torch's embedding): 2^lg lanes to a row, whose loads go four at a time, for
// rows below 16 KB (32768 x 768: float32 17.7, bf16 10.8 [16.8, 11.6]; 16384 x 2048 bf16 12.9, in the output's order
// 14.1); the output's order for longer rows, where a wave's next loads would wait for its stores (8192 x 8192:
// float32 45.8, bf16 24.3 [46.2, 25.0], by lanes 54.9 and 27.3; 8192 x 4096 float32 24.4 [24.9], 26.7), and for rows
// narrower than a piece (4000000 x 1: float32 10.9, bf16 10.0, 12.6 and 13.1).
//
// 2^lg lanes to a row. An id outside the table reads nothing and gives a row of NaN.
template <int W, typename T, typename ID>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const T* __restrict__ table, int64_t ld,
                                                        const ID* __restrict__ ids,
                                                        T* __restrict__ y, int64_t n, int vocab,
                                                        int D, float scale, int lg) {
  const int step = W << lg, c0 = W * (threadIdx.x & ((1 << lg) - 1));
  const int64_t hop = ((int64_t)gridDim.x * 256) >> lg;
  for (int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> lg; t < n; t += hop) {
    const int64_t id = (int64_t)ids[t];
    T* out = y + t * D;
    int c = c0;
    if (id < 0 || id >= vocab) {
      const float nan = __builtin_nanf("");
      for (; c < D; c += step) st_cols<W>(out + min(c, D - W), cols<W>(nan));
      continue;
    }
    const T* row = table + id * ld;
    for (; c + 3 * step + W <= D; c += 4 * step) {
      cols<W> v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = ld_cols<W>(row + c + u * step);
#pragma unroll
      for (int u = 0; u < 4; ++u) st_cols<W>(out + c + u * step, v[u] * scale);
    }
    for (; c < D; c += step) {
      const int cc = min(c, D - W);
      st_cols<W>(out + cc, ld_cols<W>(row + cc) * scale);
    }
  }
}

// A workgroup writes 256 U pieces of W columns in the output's order. `per` pieces to a row, and a piece's row by a
// reciprocal of that (i < 2^11 by per <= 2^10: the product is off by i / 2^32, less than 1 / per) or, of longer
// rows, by one comparison.
constexpr int kLookupPieces = 2;
template <int W, typename T, typename ID>
__global__ void __launch_bounds__(256) embed_order_kernel(const T* __restrict__ table, int64_t ld,
                                                          const ID* __restrict__ ids,
                                                          T* __restrict__ y, int64_t n, int vocab,
                                                          int D, float scale, int per, uint32_t inv) {
  constexpr int U = kLookupPieces, SPAN = 256 * U;
  const int64_t all = n * per;
  for (int64_t first = (int64_t)blockIdx.x * SPAN; first < all; first += (int64_t)gridDim.x * SPAN) {
    const int64_t t0 = first >> 32 ? first / per : (uint32_t)first / (uint32_t)per;   // the 64-bit division is long
    const uint32_t p0 = (uint32_t)(first - t0 * per);
    cols<W> v[U];
    int64_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = p0 + u * 256 + threadIdx.x;
      const uint32_t r = per > 1024 ? (uint32_t)(i >= (uint32_t)per) : per == 1 ? i : __umulhi(i, inv);
      const int64_t t = min(t0 + r, n - 1);
      const int c = min(W * (int)(i - r * (uint32_t)per), D - W);
      const int64_t id = (int64_t)ids[t];
      const bool ok = id >= 0 && id < vocab;
      v[u] = ld_cols<W>(table + (ok ? id : 0) * ld + c);   // of no id row 0, dropped
      v[u] = ok ? v[u] * scale : cols<W>(__builtin_nanf(""));
      at[u] = t0 + r < n ? t * D + c : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at[u] >= 0) st_cols<W>(y + at[u], v[u]);
    }
  }
}

// ---- stable sort of positions by id --------------------------------------------------------
// What sorts last and is never summed: the padding id, and ids outside the table.
template <typename ID>
__device__ __forceinline__ uint32_t sort_key(ID raw, int vocab, int64_t pad) {
  const int64_t id = (int64_t)raw;
  return id >= 0 && id < vocab && id != pad ? (uint32_t)id : (uint32_t)vocab;
}

// The lanes that hold this lane's digit, among those of `valid`.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, uint64_t valid) {
  uint64_t m = valid;
  for (int b = 0; b < bits; ++b) {
    const bool one = (digit >> b) & 1;
    const uint64_t bal = __ballot(one);
    m &= one ? bal : ~bal;
  }
  return m;
}

// The place of one key of the wave's 64: next[] holds the wave's next free place of each digit.
// Every lane of the wave calls it; an invalid lane's result means nothing.
__device__ __forceinline__ uint32_t take_place(uint32_t* next, uint32_t digit, int bits, bool ok) {
  const uint64_t peers = same_digit(digit, bits, __ballot(ok));
  const uint64_t below = peers & ((1ull << lane_id()) - 1);
  uint32_t at = 0;
  if (ok) at = next[digit];
  __builtin_amdgcn_wave_barrier();   // every lane has read before a digit's first lane adds
  if (ok && below == 0) next[digit] = at + (uint32_t)__popcll(peers);
  __builtin_amdgcn_wave_barrier();
  return at + (uint32_t)__popcll(below);
}

// Inclusive prefix sum over a wave's lanes: within the rows of 16, then their totals carried over.
template <int ctrl, int rows>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {
  v = dpp_add<0x111, 0xF>(v);   // row_shr 1, 2, 4, 8
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<0x142, 0xA>(v);   // lane 15 of each row to the next: rows 1 and 3
  v = dpp_add<0x143, 0xC>(v);   // lane 31 to rows 2 and 3
  return v;
}

// cnt[wave][digit] -> the first place of that wave's keys of that digit: digits in order, then
// waves; `before` (this thread's digit, threadIdx.x < kDigits) is what earlier workgroups hold and
// `total` what all of them do. Uses sums[kDigits / 64]; called by all kSortThreads.
__device__ __forceinline__ void digit_places(uint32_t (*cnt)[kDigits], uint32_t* sums,
                                             uint32_t before, uint32_t total) {
  const int d = threadIdx.x, wave = d >> 6;
  const uint32_t upto = wave_prefix(total);
  if (d < kDigits && (d & 63) == 63) sums[wave] = upto;
  __syncthreads();
  if (d < kDigits) {
    uint32_t at = upto - total + before;
    for (int w = 0; w < wave; ++w) at += sums[w];
    uint32_t c[kSortWaves];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) c[w] = cnt[w][d];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      cnt[w][d] = at;
      at += c[w];
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void zero_counts(uint32_t (*cnt)[kDigits]) {
  for (int i = threadIdx.x; i < kSortWaves * kDigits; i += kSortThreads) cnt[i / kDigits][i % kDigits] = 0;
}

// The share of the table that the workgroups behind the `sorters` first ones clear: 16-byte pieces
// lo .. hi - 1 of it, and with the last of them the few elements after the last piece.
struct Clear {
  f32x4* table;
  uint16_t* rest;
  int64_t lo, hi;
  int nrest;
  __device__ __forceinline__ bool operator()(int sorters) const {
    if ((int)blockIdx.x < sorters) return false;
    const int64_t hop = (int64_t)(gridDim.x - sorters) * kSortThreads;
    for (int64_t i = lo + (int64_t)(blockIdx.x - sorters) * kSortThreads + threadIdx.x; i < hi; i += hop) {
      table[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if ((int)blockIdx.x == sorters && (int)threadIdx.x < nrest) rest[threadIdx.x] = 0;
    return true;
  }
};

// Up to kSortOne tokens, by the first workgroup. Wave w holds the 64 `rounds` keys from 64 rounds w on.
template <typename ID>
__global__ void __launch_bounds__(kSortThreads) sort_one_kernel(const ID* __restrict__ ids,
                                                                uint32_t* __restrict__ keys,
                                                                uint32_t* __restrict__ pos,
                                                                const Clear clear, int n, int vocab,
                                                                int64_t pad, int passes, int bits) {
  __shared__ uint32_t cnt[kSortWaves][kDigits];
  __shared__ uint32_t sums[kDigits / 64];
  __shared__ uint32_t skey[kSortOne];
  __shared__ uint16_t spos[kSortOne];
  if (clear(1)) return;
  const int wave = threadIdx.x >> 6, lane = lane_id();
  const int rounds = (n + kSortThreads - 1) / kSortThreads;
  const int i0 = wave * rounds * 64 + lane;
  uint32_t key[kSortRounds], p[kSortRounds];
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int i = i0 + 64 * r;
    key[r] = r < rounds && i < n ? sort_key(ids[i], vocab, pad) : 0u;
    p[r] = (uint32_t)i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    const uint32_t mask = (1u << bits) - 1;
    zero_counts(cnt);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (r < rounds && i0 + 64 * r < n) atomicAdd(&cnt[wave][(key[r] >> shift) & mask], 1u);
    }
    __syncthreads();
    uint32_t total = 0;
    if (threadIdx.x < kDigits) {
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) total += cnt[w][threadIdx.x];
    }
    digit_places(cnt, sums, 0u, total);
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (r >= rounds) break;
      const bool ok = i0 + 64 * r < n;
      const uint32_t at = take_place(cnt[wave], (key[r] >> shift) & mask, bits, ok);
      if (ok && at < (uint32_t)n) {
        skey[at] = key[r];
        spos[at] = (uint16_t)p[r];
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      const int i = i0 + 64 * r;
      if (r < rounds && i < n) {
        key[r] = skey[i];
        p[r] = spos[i];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const int i = i0 + 64 * r;
    if (r < rounds && i < n) {
      keys[i] = key[r];
      pos[i] = p[r];
    }
  }
}

// More tokens: workgroup b of nb holds the `tile` keys from b tile on (tile a multiple of
// kSortThreads). First the counts of each workgroup's digits ...
template <typename ID, bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const ID* __restrict__ ids,
                                                                  const uint32_t* __restrict__ keys,
                                                                  uint32_t* __restrict__ hist,
                                                                  const Clear clear, int nb, int64_t n,
                                                                  int tile, int vocab, int64_t pad,
                                                                  int shift, int bits) {
  __shared__ uint32_t cnt[kDigits];
  if (clear(nb)) return;
  if (threadIdx.x < kDigits) cnt[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t mask = (1u << bits) - 1;
  const int64_t lo = (int64_t)blockIdx.x * tile, hi = lo + tile < n ? lo + tile : n;
  for (int64_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
    const uint32_t k = FIRST ? sort_key(ids[i], vocab, pad) : keys[i];
    atomicAdd(&cnt[(k >> shift) & mask], 1u);
  }
  __syncthreads();
  if (threadIdx.x < kDigits) hist[(int64_t)blockIdx.x * kDigits + threadIdx.x] = cnt[threadIdx.x];
}

// ... then every key to its place. Wave w of a workgroup holds tile / kSortWaves keys in a row.
template <typename ID, bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(
    const ID* __restrict__ ids, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
    uint32_t* __restrict__ okeys, uint32_t* __restrict__ opos, const uint32_t* __restrict__ hist,
    const Clear clear, int nb, int64_t n, int tile, int vocab, int64_t pad, int shift, int bits) {
  __shared__ uint32_t cnt[kSortWaves][kDigits];
  __shared__ uint32_t sums[kDigits / 64];
  if (clear(nb)) return;
  const int wave = threadIdx.x >> 6, lane = lane_id();
  const uint32_t mask = (1u << bits) - 1;
  const int share = tile / kSortWaves;
  const int64_t lo = (int64_t)blockIdx.x * tile + (int64_t)wave * share;
  zero_counts(cnt);
  __syncthreads();
  for (int r = 0; r < share; r += 64) {
    const int64_t i = lo + r + lane;
    if (i < n) {
      const uint32_t k = FIRST ? sort_key(ids[i], vocab, pad) : keys[i];
      atomicAdd(&cnt[wave][(k >> shift) & mask], 1u);
    }
  }
  uint32_t before = 0, total = 0;
  if (threadIdx.x < kDigits) {
#pragma unroll 16
    for (int b = 0; b < nb; ++b) {
      const uint32_t h = hist[(int64_t)b * kDigits + threadIdx.x];
      total += h;
      if (b < (int)blockIdx.x) before += h;
    }
  }
  __syncthreads();
  digit_places(cnt, sums, before, total);
  for (int r = 0; r < share; r += 64) {
    const int64_t i = lo + r + lane;
    const bool ok = i < n;
    uint32_t k = 0;
    if (ok) k = FIRST ? sort_key(ids[i], vocab, pad) : keys[i];
    const uint32_t at = take_place(cnt[wave], (k >> shift) & mask, bits, ok);
    if (ok && at < (uint64_t)n) {   // always, unless the ids change under the sort
      okeys[at] = k;
      opos[at] = FIRST ? (uint32_t)i : pos[i];
    }
  }
}

// ---- sums by id ------------------------------------------------------------------------------
// A wave adds the RUN sorted rows of a piece, 64 W columns of them. part (pieces, 2, D): slot 0 a
// run that came from the piece before (and may go on), slot 1 one that starts here and goes on.
template <int RUN, int W, typename T>
__global__ void __launch_bounds__(256) run_sum_kernel(const uint32_t* __restrict__ keys,
                                                      const uint32_t* __restrict__ pos,
                                                      const T* __restrict__ dy,
                                                      T* __restrict__ dtable,
                                                      float* __restrict__ part, int64_t n, int vocab,
                                                      int D, float scale, int tiles) {
  const int lane = lane_id();
  const uint32_t none = 0xffffffffu;
  const int64_t work = (n + RUN - 1) / RUN * tiles;
  for (int64_t g = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); g < work; g += (int64_t)gridDim.x * 4) {
    const int64_t piece = g / tiles;
    const int tile = (int)(g - piece * tiles);
    const int64_t i0 = piece * RUN;
    const int held = n - i0 < RUN ? (int)(n - i0) : RUN;
    uint32_t key = none, p = 0;
    if (lane < held) {
      key = keys[i0 + lane];
      p = (uint32_t)min((int64_t)pos[i0 + lane], n - 1);
    }
    const uint32_t kprev = i0 > 0 ? keys[i0 - 1] : none;
    const uint32_t knext = i0 + held < n ? keys[i0 + held] : none;
    const int rows = __popcll(__ballot(lane < held && key < (uint32_t)vocab));   // the rest sorts last
    const bool mine = W * (64 * tile + lane) < D;   // lanes past the row load its end and drop it
    const int c = min(W * (64 * tile + lane), D - W);
    cols<W> acc = 0.f;
    int from = 0;
    for (int j0 = 0; j0 < rows; j0 += 8) {
      cols<W> v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = min(j0 + u, rows - 1);
        const int64_t row = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)p, j);
        v[u] = ld_cols<W>(dy + row * D + c);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int j = j0 + u;
        if (j >= rows) break;
        acc += v[u];
        const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)key, j);
        const uint32_t kn = j + 1 < held ? (uint32_t)__builtin_amdgcn_readlane((int)key, j + 1) : knext;
        if (j + 1 < rows && kn == k) continue;
        if (mine) {
          if (from == 0 && kprev == k) st_cols<W>(part + 2 * piece * D + c, acc);
          else if (kn == k) st_cols<W>(part + (2 * piece + 1) * D + c, acc);
          else st_cols<W>(dtable + (int64_t)k * D + c, acc * scale);
        }
        acc = 0.f;
        from = j + 1;
      }
    }
  }
}

// The runs that cross pieces, each by the workgroup of the piece it starts in, 64 W columns
// (blockIdx.y): its slot 1, then slot 0 of the pieces that begin with its id. The four waves add a
// quarter of them each. Most workgroups find no such run: all that decides it is loaded at once.
template <int RUN, int W, typename T>
__global__ void __launch_bounds__(256) finish_kernel(const uint32_t* __restrict__ keys,
                                                     const float* __restrict__ part,
                                                     T* __restrict__ dtable, int64_t n, int vocab,
                                                     int D, float scale) {
  __shared__ cols<W> sums[4][64];
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const bool mine = W * (64 * (int)blockIdx.y + lane) < D;
  const int c = min(W * (64 * (int)blockIdx.y + lane), D - W);
  for (int64_t p = blockIdx.x; (p + 1) * RUN < n; p += gridDim.x) {
    // the ids before the piece, at its end, and at the start of each piece behind it
    const uint32_t before = keys[p > 0 ? p * RUN - 1 : 0], k = keys[(p + 1) * RUN - 1];
    const int64_t next = (p + 1 + lane) * RUN;
    uint32_t head = keys[next < n ? next : n - 1];
    uint64_t m = __ballot(next < n && head == k);
    if (k >= (uint32_t)vocab || !(m & 1) || (p > 0 && before == k)) continue;
    int64_t count = 1 + __popcll(m);
    while (m == ~0ull) {
      const int64_t at = (p + count + lane) * RUN;
      head = keys[at < n ? at : n - 1];
      m = __ballot(at < n && head == k);
      count += __popcll(m);
    }
    const int64_t share = (count + 3) / 4;
    const int64_t lo = wave * share, hi = lo + share < count ? lo + share : count;
    cols<W> acc = 0.f;
#pragma unroll 8
    for (int64_t i = lo; i < hi; ++i) acc += ld_cols<W>(part + (2 * (p + i) + (i == 0)) * D + c);
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && mine) {
      st_cols<W>(dtable + (int64_t)k * D + c,
                 (((acc + sums[1][lane]) + sums[2][lane]) + sums[3][lane]) * scale);
    }
    __syncthreads();
  }
}

// ---- sums by id, few tokens --------------------------------------------------------------------
// One launch without a sort: every workgroup reads all ids and lists the tokens of its own rows. Beside
// the sort (three launches and a workspace) Zipf-distributed ids of 256, D 768, float32, take 3.6 us
// against 9.7 at 64 tokens and 6.7 against 11.4 at 1024; 1024 of 50001 ids, D 1024, 29.9 against 34.6
// (7.0 TB/s). What it is slower at is a single id on all of the tokens, whose rows one workgroup of
// each slice then adds: 16.6 against 10.6 at 512, 29.6 against 12.3 at 1024. There it ends: at 2048
// Zipf's ids would gain a sixth, and the single id lose 50 us. It ends too at tables that no cache
// holds, where rows off a cache line's border are written as parts of lines (105209 x 851 float32: 94
// against 72 us sorted; in bf16, half of it, 29 against 32).
constexpr int kGatherTokens = 1024, kGatherRounds = kGatherTokens / 256;
constexpr int64_t kGatherTable = 1 << 26;   // entries
constexpr int kGatherRows = 1024;   // rows of a workgroup's, at most
constexpr int kAlone = 16;          // tokens of a row that one wave adds alone: two rounds of loads

// The rows of dy of those of hit[lo .. hi - 1] that belong to row j of the workgroup's, added in order.
template <int W, typename T>
__device__ __forceinline__ cols<W> sum_hits(const uint32_t* hit, int lo, int hi, uint32_t j,
                                            const T* __restrict__ dy, int D, int c) {
  cols<W> acc = 0.f;
  for (int i0 = lo; i0 < hi; i0 += 64) {
    const int i = i0 + lane_id();
    const uint32_t e = hit[min(i, hi - 1)];
    uint64_t m = __ballot(i < hi && e / kGatherTokens == j);
    while (m) {
      cols<W> v[8];
      int held = 0, at = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {   // past the last one its row again, not added
        if (m) {
          at = __builtin_ctzll(m);
          m &= m - 1;
          held = u + 1;
        }
        const int64_t row = (uint32_t)__builtin_amdgcn_readlane((int)e, at) % kGatherTokens;
        v[u] = ld_cols<W>(dy + row * D + c);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (u < held) acc += v[u];
      }
    }
  }
  return acc;
}

// Workgroup (b, y) owns a row of each 2^lg of the table, 64 W columns of them: its row j is row
// (b ^ j) mod 2^lg of the j-th 2^lg, so that neither neighbours (frequent ids often are) nor every 2^lg-th
// row meet in one workgroup. It lists its rows' tokens in order and clears the rows without any; a row
// of up to kAlone tokens is added by one wave, a longer one by all four, a quarter of the list each.
template <int W, typename T, typename ID>
__global__ void __launch_bounds__(256) gather_kernel(const ID* __restrict__ ids,
                                                     const T* __restrict__ dy, T* __restrict__ dtable,
                                                     int n, int vocab, int64_t pad, int D, float scale,
                                                     int lg) {
  __shared__ uint32_t hit[kGatherTokens];   // j, token
  __shared__ uint32_t count[kGatherRows];   // tokens of row j
  __shared__ int held[4];
  __shared__ cols<W> sums[4][64];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t b = blockIdx.x, mask = (1u << lg) - 1;
  const int rows = (int)(((int64_t)vocab + mask) >> lg);   // the last may lie past the table
  const bool mine = W * (64 * (int)blockIdx.y + lane) < D;
  const int c = min(W * (64 * (int)blockIdx.y + lane), D - W);
  const auto store = [&](int j, cols<W> v) {
    const int64_t id = ((int64_t)j << lg) + ((b ^ (uint32_t)j) & mask);
    if (mine && id < vocab) st_cols<W>(dtable + id * D + c, v);
  };
  for (int j = threadIdx.x; j < rows; j += 256) count[j] = 0;
  // wave w looks at kGatherTokens / 4 of the tokens from there on
  const int t0 = wave * (kGatherTokens / 4) + lane;
  uint32_t key[kGatherRounds];
  uint64_t m[kGatherRounds];
  int found = 0;
#pragma unroll
  for (int r = 0; r < kGatherRounds; ++r) {
    key[r] = t0 + 64 * r < n ? sort_key(ids[t0 + 64 * r], vocab, pad) : (uint32_t)vocab;
  }
#pragma unroll
  for (int r = 0; r < kGatherRounds; ++r) {
    m[r] = __ballot(key[r] < (uint32_t)vocab && ((key[r] ^ (key[r] >> lg)) & mask) == b);
    found += __popcll(m[r]);
  }
  if (lane == 0) held[wave] = found;
  __syncthreads();
  int at = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    at += w < wave ? held[w] : 0;
    all += held[w];
  }
  all = __builtin_amdgcn_readfirstlane(all);
#pragma unroll
  for (int r = 0; r < kGatherRounds; ++r) {
    if ((m[r] >> lane) & 1) {
      const uint32_t j = key[r] >> lg;
      hit[at + __popcll(m[r] & ((1ull << lane) - 1))] = j * kGatherTokens + t0 + 64 * r;
      atomicAdd(&count[j], 1u);
    }
    at += __popcll(m[r]);
  }
  __syncthreads();
  for (int j = wave; j < rows; j += 4) {
    if (count[j] == 0) store(j, cols<W>(0.f));
  }
  if (all == 0) return;
  int k = 0;
  for (int j0 = 0; j0 < rows; j0 += 64) {
    const uint32_t tokens = j0 + lane < rows ? count[j0 + lane] : 0;
    for (uint64_t few = __ballot(tokens > 0 && tokens <= kAlone); few; few &= few - 1, ++k) {
      if ((k & 3) != wave) continue;
      const int j = j0 + __builtin_ctzll(few);
      store(j, sum_hits<W>(hit, 0, all, j, dy, D, c) * scale);
    }
  }
  if (all <= kAlone) return;
  const int share = (all + 3) / 4, lo = wave * share, hi = min(lo + share, all);
  for (int j0 = 0; j0 < rows; j0 += 64) {
    const uint32_t tokens = j0 + lane < rows ? count[j0 + lane] : 0;
    for (uint64_t many = __ballot(tokens > kAlone); many; many &= many - 1) {
      const int j = j0 + __builtin_ctzll(many);
      const cols<W> acc = sum_hits<W>(hit, lo, hi, j, dy, D, c);
      sums[wave][lane] = acc;
      __syncthreads();
      if (wave == 0) store(j, (((acc + sums[1][lane]) + sums[2][lane]) + sums[3][lane]) * scale);
      __syncthreads();
    }
  }
}

// ---- host ------------------------------------------------------------------------------------
struct EmbedSpace {
  int64_t keys[2], pos[2], hist, part, total;   // byte offsets
  int run;                                      // sorted rows to a piece
};

static EmbedSpace embed_space(int64_t n, int64_t vocab, int64_t D) {   // for the wider of the two types, float32
  EmbedSpace s = {};
  if (n <= kGatherTokens && vocab * D <= kGatherTable) return s;   // no sort
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  for (int i = 0; i < 2; ++i) {
    s.keys[i] = take(4 * n);
    s.pos[i] = take(4 * n);
  }
  s.hist = take((int64_t)kSortBlocks * kDigits * 4);
  // the longest pieces that leave enough waves to keep HBM busy
  const int64_t tiles = D < 4 ? 1 : (D + 255) / 256;
  s.run = n * tiles >= 32 * kRunWaves ? 32 : n * tiles >= 16 * kRunWaves ? 16 : 8;
  s.part = take((n + s.run - 1) / s.run * 2 * D * 4);
  s.total = at;
  return s;
}

static bool embed_sizes_ok(int64_t n, int64_t vocab, int64_t D) {
  return n >= 0 && n < (1ll << 31) - 64 && vocab > 0 && vocab < (1ll << 31) - 1 && D > 0 && D < (1 << 22);
}

constexpr int64_t kGridMax = 1 << 20;   // workgroups of a launch: the kernels step over the rest

template <int W, typename T, typename ID>
static void launch_embed_fwd(const m3s_embed_args* a, hipStream_t s) {
  const int per = (a->width + W - 1) / W;
  const T* table = static_cast<const T*>(a->table);
  const ID* ids = static_cast<const ID*>(a->ids);
  T* y = static_cast<T*>(a->y);
  if (W == 1 || per >= 1024) {
    const uint32_t inv = per > 1 ? (uint32_t)((1ull << 32) / per + 1) : 0;
    const int64_t span = 256 * kLookupPieces, blocks = std::min(kGridMax, (a->tokens * per + span - 1) / span);
    hipLaunchKernelGGL((embed_order_kernel<W, T, ID>), dim3((unsigned)blocks), dim3(256), 0, s, table, a->table_stride,
                       ids, y, a->tokens, a->vocab, a->width, a->scale, per, inv);
    return;
  }
  if constexpr (W > 1) {
    // Lanes to a row: a wave, or as many as idle an eighth of the row's pieces less at its end (32768 rows of 768 bf16,
    // 96 pieces: 12.9 -> 10.8 us by 32 lanes; of 515, 65 pieces: 13.3 -> 10.4 by 16)
    int lg = 0;
    while (lg < 6 && (1 << lg) < per) ++lg;
    const auto idle = [&](int l) { return ((per + (1 << l) - 1) >> l << l) - per; };
    for (int l = 5; lg > 4 && l >= 4; --l) {
      if (l < lg && 8 * (idle(lg) - idle(l)) > per) lg = l;
    }
    const int64_t blocks = std::min(kGridMax, (a->tokens + (256 >> lg) - 1) / (256 >> lg));
    hipLaunchKernelGGL((embed_fwd_kernel<W, T, ID>), dim3((unsigned)blocks), dim3(256), 0, s, table, a->table_stride, ids,
                       y, a->tokens, a->vocab, a->width, a->scale, lg);
  }
}

template <int RUN, int W, typename T>
static void launch_sums(const m3s_embed_args* a, const uint32_t* keys, const uint32_t* pos, float* part,
                        hipStream_t s) {
  const int tiles = (a->width + 64 * W - 1) / (64 * W);
  const int64_t pieces = (a->tokens + RUN - 1) / RUN;
  T* dtable = static_cast<T*>(a->dtable);
  hipLaunchKernelGGL((run_sum_kernel<RUN, W, T>), dim3((unsigned)std::min(kGridMax, (pieces * tiles + 3) / 4)),
                     dim3(256), 0, s, keys, pos, static_cast<const T*>(a->dy), dtable, part, a->tokens,
                     a->vocab, a->width, a->scale, tiles);
  if (pieces < 2) return;   // nothing to cross
  hipLaunchKernelGGL((finish_kernel<RUN, W, T>), dim3((unsigned)std::min(kGridMax, pieces - 1), (unsigned)tiles),
                     dim3(256), 0, s, keys, part, dtable, a->tokens, a->vocab, a->width,
                     a->scale);
}

template <int W, typename T, typename ID>
static void launch_embed_bwd(const m3s_embed_args* a, hipStream_t s) {
  const int64_t n = a->tokens;
  const ID* ids = static_cast<const ID*>(a->ids);
  const T* dy = static_cast<const T*>(a->dy);
  T* dtable = static_cast<T*>(a->dtable);
  const EmbedSpace sp = embed_space(n, a->vocab, a->width);
  if (sp.total == 0) {
    int lg = 0;   // 1024 workgroups to a slice, four to a CU: more would each read the ids again
    while (lg < 10 && (1 << lg) < a->vocab) ++lg;
    while (((int64_t)kGatherRows << lg) < a->vocab) ++lg;
    hipLaunchKernelGGL((gather_kernel<W, T, ID>), dim3(1u << lg, (a->width + 64 * W - 1) / (64 * W)), dim3(256), 0, s,
                       ids, dy, dtable, (int)n, a->vocab, a->padding_idx, a->width, a->scale, lg);
    return;
  }
  char* w = static_cast<char*>(a->workspace);
  const auto u32 = [&](int64_t off) { return reinterpret_cast<uint32_t*>(w + off); };
  int width = 1;   // bits of a key: 0 .. vocab
  while ((uint64_t)a->vocab >> width) ++width;
  const int passes = (width + kDigitBits - 1) / kDigitBits, bits = (width + passes - 1) / passes;
  // each launch of the sort clears an equal share of the table
  const int64_t bytes = (int64_t)a->vocab * a->width * sizeof(T), pieces = bytes / 16;
  const int shares = n <= kSortOne ? 1 : 2 * passes;
  const auto clear = [&](int share) {
    Clear c;
    c.table = static_cast<f32x4*>(a->dtable);
    c.rest = reinterpret_cast<uint16_t*>(static_cast<char*>(a->dtable) + pieces * 16);
    c.lo = pieces * share / shares;
    c.hi = pieces * (share + 1) / shares;
    c.nrest = share + 1 == shares ? (int)((bytes - pieces * 16) / 2) : 0;
    return c;
  };
  // Workgroups: a piece to a thread, and no loop (the gradient of one token of 131072 x 1536 float32 takes 135 us
  // so, 144 with 8 pieces or more to a thread of up to 8192; of 100 tokens of 256000 x 2048 341 and 391).
  const auto cleaners = [&](const Clear& c) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(kGridMax, (c.hi - c.lo + kSortThreads - 1) / kSortThreads));
  };
  int last = 0;
  if (n <= kSortOne) {
    const Clear c = clear(0);
    hipLaunchKernelGGL((sort_one_kernel<ID>), dim3(1 + cleaners(c)), dim3(kSortThreads), 0, s, ids,
                       u32(sp.keys[0]), u32(sp.pos[0]), c, (int)n, a->vocab, a->padding_idx, passes, bits);
  } else {
    // the fewest 1024-key rounds that leave at most kSortBlocks workgroups
    const int64_t rounds = (n + (int64_t)kSortThreads * kSortBlocks - 1) / ((int64_t)kSortThreads * kSortBlocks);
    const int tile = (int)(rounds * kSortThreads);
    const int nb = (int)((n + tile - 1) / tile);
    for (int p = 0; p < passes; ++p) {
      const int from = (p + 1) & 1, to = p & 1;
      uint32_t *ik = u32(sp.keys[from]), *ip = u32(sp.pos[from]), *ok = u32(sp.keys[to]), *op = u32(sp.pos[to]);
      const Clear c0 = clear(2 * p), c1 = clear(2 * p + 1);
      const auto go = [&](auto count, auto place) {
        hipLaunchKernelGGL(count, dim3(nb + cleaners(c0)), dim3(kSortThreads), 0, s, ids, ik, u32(sp.hist), c0,
                           nb, n, tile, a->vocab, a->padding_idx, p * bits, bits);
        hipLaunchKernelGGL(place, dim3(nb + cleaners(c1)), dim3(kSortThreads), 0, s, ids, ik, ip, ok, op,
                           u32(sp.hist), c1, nb, n, tile, a->vocab, a->padding_idx, p * bits, bits);
      };
      if (p == 0) go(sort_count_kernel<ID, true>, sort_place_kernel<ID, true>);
      else go(sort_count_kernel<ID, false>, sort_place_kernel<ID, false>);
      last = to;
    }
  }
  if (n == 0) return;
  const uint32_t *keys = u32(sp.keys[last]), *pos = u32(sp.pos[last]);
  float* part = reinterpret_cast<float*>(w + sp.part);
  if (sp.run == 32) launch_sums<32, W, T>(a, keys, pos, part, s);
  else if (sp.run == 16) launch_sums<16, W, T>(a, keys, pos, part, s);
  else launch_sums<8, W, T>(a, keys, pos, part, s);
}

template <typename T, typename ID>
static void launch_embed(const m3s_embed_args* a, hipStream_t s, bool bwd) {
  const bool narrow = a->width < kCols<T>;
  // sums of rows up to 256 wide: four columns of bf16 a lane, or half the lanes of a wave would idle
  if (bwd && !narrow && a->width <= 256) launch_embed_bwd<4, T, ID>(a, s);
  else if (bwd) narrow ? launch_embed_bwd<1, T, ID>(a, s) : launch_embed_bwd<kCols<T>, T, ID>(a, s);
  else narrow ? launch_embed_fwd<1, T, ID>(a, s) : launch_embed_fwd<kCols<T>, T, ID>(a, s);
}

static void dispatch_embed(const m3s_embed_args* a, hipStream_t s, bool bwd) {
  const bool wide = a->id_bytes == 8;
  if (a->dtype == M3S_DTYPE_BF16) wide ? launch_embed<bf16, int64_t>(a, s, bwd) : launch_embed<bf16, int32_t>(a, s, bwd);
  else wide ? launch_embed<float, int64_t>(a, s, bwd) : launch_embed<float, int32_t>(a, s, bwd);
}

static int32_t check_embed(const m3s_embed_args* a, const char* who, bool bwd) {
  M3S_REQUIRE(a != nullptr, "%s: args is NULL", who);
  M3S_REQUIRE(a->struct_size == (int32_t)sizeof(m3s_embed_args),
              "%s: struct_size %d != %d (ABI mismatch)", who, a->struct_size,
              (int)sizeof(m3s_embed_args));
  M3S_REQUIRE(a->dtype == M3S_DTYPE_BF16 || a->dtype == M3S_DTYPE_F32, "%s: bad dtype", who);
  M3S_REQUIRE(a->id_bytes == 4 || a->id_bytes == 8, "%s: ids of %d bytes, must be 4 or 8", who, a->id_bytes);
  M3S_REQUIRE(embed_sizes_ok(a->tokens, a->vocab, a->width),
              "%s: bad sizes (tokens %lld, vocab %d, width %d)", who, (long long)a->tokens, a->vocab, a->width);
  const uintptr_t es = a->dtype == M3S_DTYPE_BF16 ? 2 : 4;
  M3S_REQUIRE((uintptr_t)a->ids % a->id_bytes == 0, "%s: ids misaligned", who);
  if (!bwd) {
    if (a->tokens == 0) return 0;
    M3S_REQUIRE(a->ids && a->table && a->y, "%s: NULL pointer", who);
    M3S_REQUIRE((uintptr_t)a->table % es == 0 && (uintptr_t)a->y % es == 0, "%s: misaligned rows", who);
    M3S_REQUIRE(a->table_stride >= 0, "%s: negative table stride", who);
    return 0;
  }
  M3S_REQUIRE(a->dtable && (a->tokens == 0 || (a->ids && a->dy)), "%s: NULL pointer", who);
  M3S_REQUIRE((uintptr_t)a->dy % es == 0, "%s: misaligned rows", who);
  M3S_REQUIRE(aligned16(a->workspace) && aligned16(a->dtable), "%s: dtable and workspace must be 16-byte aligned", who);
  const int64_t need = embed_space(a->tokens, a->vocab, a->width).total;   // none for few tokens
  M3S_REQUIRE(need == 0 || a->workspace, "%s: NULL pointer", who);
  M3S_REQUIRE(a->workspace_bytes >= need, "%s: workspace of %lld bytes, needs %lld", who,
              (long long)a->workspace_bytes, (long long)need);
  return 0;
}

}  // namespace m3s

using namespace m3s;

extern "C" int64_t m3s_embed_bwd_workspace_bytes(int64_t tokens, int32_t vocab, int32_t width) {
  if (!embed_sizes_ok(tokens, vocab, width)) return -1;
  return embed_space(tokens, vocab, width).total;
}

extern "C" int32_t m3s_embed_fwd(const m3s_embed_args* a, void* stream) {
  clear_error();
  if (int32_t rc = check_embed(a, "m3s_embed_fwd", false)) return rc;
  if (a->tokens == 0) return 0;
  dispatch_embed(a, static_cast<hipStream_t>(stream), false);
  return launch_status("m3s_embed_fwd");
}

extern "C" int32_t m3s_embed_bwd(const m3s_embed_args* a, void* stream) {
  clear_error();
  if (int32_t rc = check_embed(a, "m3s_embed_bwd", true)) return rc;
  dispatch_embed(a, static_cast<hipStream_t>(stream), true);
  return launch_status("m3s_embed_bwd");
}
