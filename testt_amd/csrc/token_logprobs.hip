// Log probabilities of given tokens, the entropy of their distributions and the top alternatives,
// from logits, and the gradient of the logits.
//
// Per row of logits z, temperature T, with m = max z, d = (z - m) / T, S = sum exp(d):
//   logprob = d[token] - ln S        entropy = ln S - sum(exp(d) d) / S
//   top alternatives: the K largest z, equal ones by the lower column, each with d - ln S
//   dz = (1/T) [ g_lp (1[token] - p) + sum_k g_k (1[id_k] - p) - g_ent p (ln p + entropy) ]
// Everything is taken relative to the row's maximum, so masks of the type's lowest value and -inf
// cost no precision (a masked column has p = 0 and adds nothing).  A NaN or +inf in a row makes its
// numbers NaN; a NaN ranks with -inf among the alternatives.
//
// Forward: one pass over the logits.  A workgroup reads a part of a row (a whole row when there are
// many rows) in steps of one 16-byte chunk per thread and keeps, per lane, the running maximum, the
// sum of exponentials and of exponentials times their argument, rescaled when the maximum rises.
//
// The alternatives come out of the same pass.  Each thread knows the largest value it has seen; the K-th
// largest of 64 groups' maxima is a bound: K columns at least as large have been seen, all of them
// further left than what is still to come, so from there on only a value strictly above the bound can be
// among the K, and its chunk's number goes into a short list in LDS.  The bound is raised after 1, 4,
// 16, 64 ... steps, so the list stays at some ten times K entries whatever the row's length.  Of the first
// step's columns, those equal to its bound are listed by themselves, only as far as they can count (by
// their order).  At the end the listed chunks that reach the last bound are read again, and their
// columns ranked.  Where the list overflows (a row that rises from left to right) the row is read once
// more by the last bound: 1030 rows of 40000 fp32 columns with 32 alternatives take 83 us instead of 39,
// of 151936 columns 271 instead of 115 (K searches instead: 2118 and 10924).  Where even those columns do
// not fit (large ones that come back every 1024 columns, in some of the threads' places alone), the row
// is ranked by K searches.
//
// Few rows are cut into parts, whose statistics and alternatives a second launch joins.
//
// Measured (MI355X): 2048 rows of 151936 bf16 (622 MB) 100 us without alternatives (6.2 TB/s; reading
// alone 93), 107 with 8, 118 with 32: the bounds and lists are latency between barriers that all the
// rows of a CU meet together, so 512 threads a row (127 us with 8 where 256 took 115) and 1024 are slower, and
// fewer or more loads in flight change nothing.  The gradient of 888 rows fp16 reads and writes 540 MB in
// 77 us (7.0 TB/s, its reads in part from the Infinity Cache, where the forward left the rows; 91 behind a
// forward that streams past them, where one 16-byte store a thread took 114 and eight 99).

#include <algorithm>
#include <type_traits>

#include "elem.hpp"

namespace soupk {
namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / kWave;
constexpr int kGroup = kLpThreads / 64;   // neighbouring threads whose largest value bounds the list
constexpr int kLpUnroll = 4;              // chunk loads in flight per thread
constexpr int kGradThreads = 256, kGradUnroll = 4;
constexpr int kMaxTop = 32;
// Workgroups per CU that parts of rows are cut for, to the nearest whole number a row (151936 fp16 columns
// without alternatives: 200 rows 16.9 us in 5 parts, 17.9 in 6; 888 rows 48.6 whole, 51.5 in 2).  With
// alternatives, where a part costs its bounds and lists, three: 333 rows of 32003 fp32 columns with five
// 23.8 us, 25.4 cut for four a CU; 300 rows of 151936 bf16 with eight 32.9, 35.0 cut for two.
constexpr int kLpFill = 4, kLpFillTop = 3;
constexpr int kListCap = 1024;        // chunks that a part lists
constexpr int kKeepCap = 1280;        // columns that it ranks
constexpr int kMaxParts = 64;
constexpr int64_t kIgnored = -100;
constexpr float kFloor = -200.f;      // below 2^kFloor an exponential is zero in fp32

// Rows of the logits: row r is (r / inner, r % inner) with its two strides (elements).
struct LpRows {
  int64_t inner, stride_outer, stride_inner, V, count;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    const int64_t o = r / inner;
    return o * stride_outer + (r - o * inner) * stride_inner;
  }
};

// A 16-byte chunk: 8 half-size or 4 fp32 columns, and the order of its type's values as integers
// (kBits of them; a NaN as -inf, -0 as 0).
template <typename T>
struct Chunk {
  static constexpr int N = 16 / Elem<T>::kBytes;
  static constexpr int kBits = 8 * Elem<T>::kBytes;
  u32x4 w;
  // base: uniform; off: bytes
  template <bool NT>
  __device__ __forceinline__ void load(const char* base, uint32_t off) {
    w = ld16<NT>(base + off);
  }
  __device__ __forceinline__ void unpack(float* v) const {
    if constexpr (std::is_same_v<T, float>) {
      const f32x4 f = __builtin_bit_cast(f32x4, w);
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
      Elem<T>::unpack8(typename Elem<T>::Raw8{w}, v);
    }
  }
  // x = z c + add, fused.  (fp16 columns from the loaded words, which lets the instruction that widens
  // one operand do it: 2048 rows of 151936 102.9 -> 99.7 us against the columns unpacked before.)
  __device__ __forceinline__ void scale(float* x, float c, float add) const {
    if constexpr (std::is_same_v<T, f16>) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f16x2 h = as_h2(w[q]);
        x[2 * q] = __builtin_fmaf(static_cast<float>(h[0]), c, add);
        x[2 * q + 1] = __builtin_fmaf(static_cast<float>(h[1]), c, add);
      }
    } else {
      float v[N];
      unpack(v);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = __builtin_fmaf(v[j], c, add);
    }
  }
  // Columns of -inf.
  __device__ __forceinline__ void clear() {
    const uint32_t inf = kBits == 32 ? 0xff800000u
                                     : std::is_same_v<T, f16> ? 0xfc00fc00u : 0xff80ff80u;
    w = u32x4{inf, inf, inf, inf};
  }
  // The largest column, NaN passed over.
  __device__ __forceinline__ float max() const {
    if constexpr (std::is_same_v<T, f16>) {
      const f16x2 m = __builtin_elementwise_max(
          __builtin_elementwise_max(as_h2(w.x), as_h2(w.y)),
          __builtin_elementwise_max(as_h2(w.z), as_h2(w.w)));
      return static_cast<float>(__builtin_elementwise_max(m[0], m[1]));
    } else {
      float v[N];
      unpack(v);
      float m = v[0];
#pragma unroll
      for (int j = 1; j < N; ++j) m = fmaxf(m, v[j]);
      return m;
    }
  }
  static __device__ __forceinline__ void store(char* p, const float* v) {
    if constexpr (std::is_same_v<T, float>)
      st16<true>(p, __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}));
    else
      Elem<T>::template store8<true>(p, v);
  }
  static __device__ __forceinline__ uint32_t key(float z) {
    if (z != z) z = -INFINITY;
    uint32_t b = z == 0.f ? 0u : __builtin_bit_cast(uint32_t, z);
    if constexpr (std::is_same_v<T, f16>)
      b = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<f16>(z == 0.f ? 0.f : z)))
          << 16;
    b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return b >> (32 - kBits);
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    uint32_t b = k << (32 - kBits);
    b = (b & 0x80000000u) ? b & 0x7fffffffu : ~b;
    if constexpr (std::is_same_v<T, f16>) return h2f(b >> 16);
    else if constexpr (std::is_same_v<T, bf16>) return bf2f(b >> 16);
    else return __builtin_bit_cast(float, b);
  }
};

// Running statistics: the maximum m, S = sum 2^x and A = sum 2^x x over x = z c - m c, c = log2(e) / T.
// x is one fused multiply-add with the rounded m c: its rounding, the shift m c - round(m c), is in all x of
// one m alike, so it drops out of differences and of ln S once it is taken off there.  Up to |m c| = 2^20 it
// is 2^-5 at most; it grows with m c (to 2^7 from 2^31 on, where 2^x overflows).  Beyond that (rows far from
// zero beside the temperature, masks of -1e9, of the lowest value or -inf alone, +inf) x is (z - m) c, with no
// shift.
struct Stats {
  float m, s, a;
};

__device__ __forceinline__ bool plain_form(float mc) { return fabsf(mc) < 0x1p20f; }
__device__ __forceinline__ float exponent(float z, float m, float mc, float c) {
  return plain_form(mc) ? __builtin_fmaf(z, c, -mc) : (m == -INFINITY ? z : z - m) * c;
}
// What every x relative to m is above (z - m) c.
__device__ __forceinline__ float shift_of(float m, float mc, float c) {
  return plain_form(mc) ? __builtin_fmaf(m, c, -mc) : 0.f;
}

// The statistics relative to another maximum m >= st.m.
__device__ __forceinline__ void move_max(Stats& st, float m, float c) {
  if (st.m == m) return;
  const float from = st.m * c, to = m * c;
  // (one of them out of the plain form: the shift of the other does not cancel)
  float x = plain_form(from) && plain_form(to)
                ? from - to
                : (st.m - m) * c + (shift_of(m, to, c) - shift_of(st.m, from, c));
  x = fmaxf(x, kFloor);
  const float f = st.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x);   // (then s and a are 0)
  st.a = f * __builtin_fmaf(x, st.s, st.a);
  st.s = f * st.s;
  st.m = m;
}

// While a lane reads, its m may lag behind the largest value by kLag of x (2^8 in the terms): moving it
// costs an exponential and a branch that some lane of 64 takes at nearly every chunk of a row of 40 or 80
// chunks a lane.  The maximum itself is kept beside it, and the statistics are moved to it at the end. (A's terms
// are then up to 8 larger, which adds 8 roundings of S, 2^-21 of the entropy's unit, at most.)  2048 rows of
// 151936 bf16 102.7 -> 99.2 us.
constexpr float kLag = 8.f;

// A column by itself, as absorb takes them.
struct OneColumn {
  static constexpr int N = 1;
  float z;
  __device__ __forceinline__ void unpack(float* v) const { *v = z; }
  __device__ __forceinline__ void scale(float* x, float c, float add) const {
    *x = __builtin_fmaf(z, c, add);
  }
};

// Folds columns with maximum bm into the statistics; the whole wavefront calls it.  limit: st.m and
// the lag; odd: a lane's m is out of the plain form's range (both kept across calls).  A column of -inf makes the sum A NaN (0 * -inf): then A is formed again with the exponents
// bounded.
template <typename W>
__device__ __forceinline__ void absorb(Stats& st, float& mc, float& limit, bool& odd, const W& w,
                                       float bm, float c, float lag) {
  constexpr int N = W::N;
  if (__any(bm > limit)) {
    const float m = bm > limit ? bm : st.m, to = m * c;
    const bool far = __any(!plain_form(to));
    if (odd || far) {
      move_max(st, m, c);
    } else {                                       // (a lane that stays: times 1)
      const float x = fmaxf(mc - to, kFloor), f = __builtin_amdgcn_exp2f(x);
      st.a = f * __builtin_fmaf(x, st.s, st.a);
      st.s = f * st.s;
      st.m = m;
    }
    mc = to;
    limit = m + lag;
    odd = far;
  }
  float e[N], x[N];
  if (!odd) {
    w.scale(x, c, -mc);
  } else {
    w.unpack(x);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = exponent(x[j], st.m, mc, c);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) e[j] = __builtin_amdgcn_exp2f(x[j]);
  float s = e[0], a = e[0] * x[0];
#pragma unroll
  for (int j = 1; j < N; ++j) {
    s = s + e[j];
    a = __builtin_fmaf(e[j], x[j], a);
  }
  if (a != a) {
    a = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) a = __builtin_fmaf(e[j], fmaxf(x[j], kFloor), a);
  }
  st.s = st.s + s;
  st.a = st.a + a;
}

struct Cand {
  uint32_t key;   // Chunk<T>::key of the value
  uint32_t col;
};
__device__ __forceinline__ bool ahead(const Cand& a, const Cand& b) {
  return a.key > b.key || (a.key == b.key && a.col < b.col);
}
constexpr uint32_t kNoCol = 0xffffffffu;     // an entry past the last candidate

// What a part hands on.
struct PartOut {
  Stats* stats;     // [rows, parts]
  Cand* cand;       // [rows, parts, K], best first
};
struct RowOut {
  float *logprob, *entropy, *row_max, *row_sum, *top_lp;
  int64_t* top_id;
};

struct ListLds {
  // First kListCap: chunks (the key of their largest column, their number in the part); then the columns
  // that are ranked at the end.  (The join ranks from the whole.)
  Cand list[kListCap + kKeepCap];
  Cand tie[kMaxTop];            // the leftmost columns that equal a bound
  uint32_t group_max[64];
  unsigned long long group_best[64];
  int count, kept, ties;
  int wave_n[kLpWaves];
  Cand best[kLpWaves];
  Cand top[kMaxTop];
};

// The K-th largest of the 64 groups' largest keys, by two bits a step; every thread of the workgroup
// calls it and gets it.
template <int BITS>
__device__ __forceinline__ uint32_t raise_bound(ListLds& s, uint32_t k, int K) {
  const int lane = threadIdx.x & 63;
  k = max(k, static_cast<uint32_t>(dpp_i<kDppQuad1032>(static_cast<int>(k))));
  k = max(k, static_cast<uint32_t>(dpp_i<kDppQuad2301>(static_cast<int>(k))));
  static_assert(kGroup == 4, "a group is a DPP quad");
  __syncthreads();                               // (group_max of the last call has been read)
  if (threadIdx.x % kGroup == 0) s.group_max[threadIdx.x / kGroup] = k;
  __syncthreads();
  const uint32_t mine = s.group_max[lane];
  uint32_t bound = 0;
#pragma unroll
  for (int b = BITS - 2; b >= 0; b -= 2) {
    const uint32_t c1 = bound | (1u << b), c2 = bound | (2u << b), c3 = bound | (3u << b);
    const int n1 = __popcll(__ballot(mine >= c1)), n2 = __popcll(__ballot(mine >= c2)),
              n3 = __popcll(__ballot(mine >= c3));
    bound = n3 >= K ? c3 : n2 >= K ? c2 : n1 >= K ? c1 : bound;
  }
  return bound;
}

__device__ __forceinline__ void push(ListLds& s, uint32_t key, uint32_t chunk) {
  const int at = atomicAdd(&s.count, 1);
  if (at < kListCap) s.list[at] = Cand{key, chunk};
}
__device__ __forceinline__ void keep(ListLds& s, uint32_t key, uint32_t col) {
  const int at = atomicAdd(&s.kept, 1);
  if (at < kKeepCap) s.list[kListCap + at] = Cand{key, col};
}

// Sum of the lanes up to and including this one.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
  v = row16_max(v);
  return fmaxf(fmaxf(lanef(v, 0), lanef(v, 16)), fmaxf(lanef(v, 32), lanef(v, 48)));
}

// Lists longer than this are thinned before they are ranked, which takes a list's length squared: few
// columns (64 rows of 600 fp16 with 20 alternatives 75.7 us ranked whole, 10.4 thinned), or many equal ones at the bound.
constexpr int kRankAll = 128;

// Leaves of n > kRankAll candidates those that are not behind the K-th best of the 64 groups' best ones, in
// place; returns how many.  (With more than 128 entries 32 groups have one.)
__device__ int thin_list(ListLds& s, Cand* list, int n, int K) {
  const int tid = threadIdx.x;
  auto order = [](const Cand& c) {
    return static_cast<unsigned long long>(c.key) << 32 | static_cast<uint32_t>(~c.col);
  };
  unsigned long long best = 0;
#pragma unroll 1
  for (int i = tid; i < n; i += kLpThreads) best = max(best, order(list[i]));
  best = max(best, __shfl_xor(best, 1));
  best = max(best, __shfl_xor(best, 2));
  __syncthreads();                               // (n, the list's count, has been read)
  if (tid % kGroup == 0) s.group_best[tid / kGroup] = best;
  if (tid == 0) s.kept = 0;
  __syncthreads();
  best = s.group_best[tid & 63];
  int rank = 0;
#pragma unroll 4
  for (int j = 0; j < 64; ++j) rank += s.group_best[j] > best ? 1 : 0;
  const int at = __builtin_ctzll(__ballot(rank == K - 1));       // (the groups' best ones differ)
  const unsigned long long bound = s.group_best[at];
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kLpThreads) {
    const bool on = i0 + tid < n;
    const Cand c = on ? list[i0 + tid] : Cand{0, kNoCol};
    __syncthreads();                             // (the places up to here are free)
    if (on && order(c) >= bound) list[atomicAdd(&s.kept, 1)] = c;
  }
  __syncthreads();
  return s.kept;
}

// Writes the K best of n candidates in order (entries past the last one have column kNoCol); every
// thread of the workgroup calls it.
__device__ __forceinline__ void rank_list(ListLds& s, Cand* list, int n, int K, Cand* out) {
  if (n > kRankAll) n = thin_list(s, list, n, K);
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const Cand mine = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += ahead(list[j], mine) ? 1 : 0;
    if (rank < K) out[rank] = mine;
  }
  for (int i = n + threadIdx.x; i < K; i += kLpThreads) out[i] = Cand{0, kNoCol};
}

// The K best columns of [col0, col1) by K searches, each for the best one behind the last.
template <typename T>
__device__ void search_top(ListLds& s, const char* row, int64_t col0, int64_t col1, int K) {
  Cand last{0xffffffffu, 0};
  bool any = true;
  for (int k = 0; k < K; ++k) {
    Cand best{0, kNoCol};
    if (any)
      for (int64_t i = col0 + threadIdx.x; i < col1; i += kLpThreads) {
        const Cand c{Chunk<T>::key(Elem<T>::load1(row + i * Elem<T>::kBytes)),
                     static_cast<uint32_t>(i)};
        if ((k == 0 || ahead(last, c)) && ahead(c, best)) best = c;
      }
    for (int d = 32; d > 0; d >>= 1) {
      const Cand o{__shfl_xor(best.key, d), __shfl_xor(best.col, d)};
      if (ahead(o, best)) best = o;
    }
    if ((threadIdx.x & 63) == 0) s.best[threadIdx.x >> 6] = best;
    __syncthreads();
    best = s.best[0];
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w)
      if (ahead(s.best[w], best)) best = s.best[w];
    if (threadIdx.x == 0) s.top[k] = best;
    any = best.col != kNoCol;
    last = best;
    __syncthreads();
  }
}

// Lists the columns of a step that equal `bound`, as far as they are among the first K of them from the
// left, `before` of them lying in earlier steps; returns how many the step holds.  The whole workgroup
// calls it; on: the thread has a chunk, of columns from col on.
template <typename T>
__device__ __forceinline__ int list_ties(ListLds& s, const Chunk<T>& chunk, bool on, uint32_t col,
                                         uint32_t bound, int K, int before) {
  constexpr int N = Chunk<T>::N;
  const int wave = threadIdx.x >> 6;
  uint32_t equal = 0;                            // a bit for each column
  if (on) {
    float z[N];
    chunk.unpack(z);
#pragma unroll
    for (int j = 0; j < N; ++j) equal |= Chunk<T>::key(z[j]) == bound ? 1u << j : 0u;
  }
  const int own = __popc(equal);
  const int upto = wave_scan(own);               // equal columns left of and in this thread's
  if ((threadIdx.x & 63) == 63) s.wave_n[wave] = upto;
  __syncthreads();
  int left = before + upto - own, total = 0;
  for (int k = 0; k < kLpWaves; ++k) {
    left += k < wave ? s.wave_n[k] : 0;
    total += s.wave_n[k];
  }
  for (; equal != 0 && left < K; equal &= equal - 1, ++left) {
    s.tie[left] = Cand{bound, col + static_cast<uint32_t>(__builtin_ctz(equal))};
    atomicAdd(&s.ties, 1);
  }
  return total;
}

// The lists of a part once more, by a bound that holds for all of it: every chunk with a column above it
// and the leftmost columns that equal it.
template <typename T>
__device__ void list_again(ListLds& s, const char* base, int n, uint32_t col_base, uint32_t key,
                           int K) {
  using C = Chunk<T>;
  __syncthreads();                               // (the first lists have been counted)
  if (threadIdx.x == 0) s.count = s.ties = 0;
  const float bound = C::value(key);
  int ties = 0;
  for (int i0 = 0; i0 < n; i0 += kLpThreads) {
    const int i = i0 + static_cast<int>(threadIdx.x);
    const bool on = i < n;
    C w;
    w.template load<false>(base, on ? static_cast<uint32_t>(i) * 16u : 0u);
    __syncthreads();                             // (wave_n and the cleared counts)
    if (ties < K)
      ties += list_ties<T>(s, w, on, col_base + static_cast<uint32_t>(i) * C::N, key, K, ties);
    const float bm = w.max();
    if (on && bm > bound) push(s, C::key(bm), static_cast<uint32_t>(i));
  }
  __syncthreads();
}

// Statistics of the workgroup, in every thread.
__device__ __forceinline__ Stats merge_stats(Stats* lds, Stats st, float c) {
  move_max(st, wave_max(st.m), c);
  st.s = wave_sum(st.s);
  st.a = wave_sum(st.a);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = st;
  __syncthreads();
  float mx = lds[0].m;
#pragma unroll
  for (int w = 1; w < kLpWaves; ++w) mx = fmaxf(mx, lds[w].m);
  Stats r{mx, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    Stats p = lds[w];
    move_max(p, mx, c);
    r.s = r.s + p.s;
    r.a = r.a + p.a;
  }
  return r;
}

// ln S of a row relative to its maximum: the sum's logarithm without the rounding of m c that the
// exponents share (NaN for a row of -inf alone, as the formula gives); a column's log probability.
__device__ __forceinline__ float log_sum(const Stats& st, float c) {
  if (!(st.m > -INFINITY)) return NAN;
  return logf(st.s) - kLn2 * shift_of(st.m, st.m * c, c);
}
template <typename T>
__device__ __forceinline__ float column_lp(const char* row, int64_t col, const Stats& st,
                                           float inv_t, float lse) {
  const float z = Elem<T>::load1(row + col * Elem<T>::kBytes);
  return (z - st.m) * inv_t - lse;
}

// The numbers of a row from its statistics (one thread).
template <typename T>
__device__ __forceinline__ void write_row(const RowOut& o, int64_t r, const Stats& st,
                                          const char* row, int64_t V, int64_t tok, float inv_t,
                                          float lse) {
  // (the exponents' shared rounding is in both terms)
  o.entropy[r] = (st.m > -INFINITY ? logf(st.s) : NAN) - kLn2 * (st.a / st.s);
  float lp = NAN;
  if (tok == kIgnored) lp = 0.f;
  else if (tok >= 0 && tok < V) lp = column_lp<T>(row, tok, st, inv_t, lse);
  o.logprob[r] = lp;
  if (o.row_max != nullptr) {
    o.row_max[r] = st.m;
    o.row_sum[r] = st.s;
  }
}

// KEEP: the rows are read through the caches, for the backward that comes back to them (888 rows of
// 151936 forward + backward 141.4 -> 131.4 us, 200 rows 41.4 -> 38.2, 2048 rows 312 -> 306); without one
// they stream past (the forward of 888 rows alone 48.6 us, through the caches 53.8).
// Eight workgroups a CU (registers by the launch bound, the lists below 20 KB): with the seven that fit
// otherwise, eight alternatives of 1792 bf16 rows took 106.3 us instead of 95.6, of 2048 rows 113.8
// instead of 106.4.
template <typename T, bool TOP, bool KEEP>
__global__ __launch_bounds__(kLpThreads, 8) void token_logprobs_kernel(
    const char* __restrict__ logits, const int64_t* __restrict__ tokens, LpRows rows, float c,
    float inv_t, int K, int parts, int64_t part_chunks, int64_t r0, PartOut part, RowOut out) {
  using C = Chunk<T>;
  constexpr int N = C::N;
  constexpr int kSize = Elem<T>::kBytes;
  __shared__ Stats stat_lds[kLpWaves];
  __shared__ std::conditional_t<TOP, ListLds, int> lds;
  const int64_t r = r0 + blockIdx.x / static_cast<uint32_t>(parts);
  const int which = static_cast<int>(blockIdx.x % static_cast<uint32_t>(parts));
  const char* const row = logits + rows.at(r) * kSize;
  const int64_t chunks = rows.V / N;
  const int64_t first = which * part_chunks;
  const int64_t last = min(chunks, first + part_chunks);
  const int tid = threadIdx.x;
  Stats st{-INFINITY, 0.f, 0.f};
  float mc = -INFINITY, limit = -INFINITY;
  const float lag = kLag / c;
  bool odd = true;
  float tmax = -INFINITY;        // this thread's largest value so far (never NaN)
  float bound = -INFINITY;
  uint32_t first_key = 0;        // the first step's bound
  if constexpr (TOP) {
    if (tid == 0) lds.count = lds.kept = lds.ties = 0;
    __syncthreads();
  }
  // Offsets within the part fit 32 bits (the host cuts longer rows).
  const char* const base = row + first * 16;
  const int n = static_cast<int>(last - first);          // (<= 0: an empty last part)
  const int steps = n > 0 ? (n + kLpThreads - 1) / kLpThreads : 0;
  const uint32_t col_base = static_cast<uint32_t>(first) * N;
  int next_raise = kLpUnroll;
  for (int step = 0; step < steps; step += kLpUnroll) {
    C w[kLpUnroll];
    const int i0 = step * kLpThreads + tid;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      // (past the part's end: its first chunk, so that no load waits for a branch ...)
      const int i = i0 + u * kLpThreads;
      w[u].template load<!KEEP>(base, i < n ? static_cast<uint32_t>(i) * 16u : 0u);
    }
    if constexpr (TOP) {
      if (step == next_raise) {
        next_raise *= 4;
        bound = C::value(raise_bound<C::kBits>(lds, C::key(tmax), K));
      }
    }
    if ((step + kLpUnroll) * kLpThreads > n) {
      // (... and counted as -inf)
#pragma unroll
      for (int u = 0; u < kLpUnroll; ++u)
        if (i0 + u * kLpThreads >= n) w[u].clear();
    }
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      if (step + u >= steps) break;              // (888 rows of 151936 fp16 54.2 -> 52.4 us)
      const int i = i0 + u * kLpThreads;
      const float bm = w[u].max();
      absorb(st, mc, limit, odd, w[u], bm, c, lag);
      tmax = fmaxf(tmax, bm);
      if constexpr (TOP) {
        if (u == 0 && step == 0) {
          // The first step's columns against the bound that they give: the chunks with one above it,
          // and as many of the equal ones, from the left, as the K can still take.
          first_key = raise_bound<C::kBits>(lds, C::key(tmax), K);
          bound = C::value(first_key);
          list_ties<T>(lds, w[u], i < n, col_base + static_cast<uint32_t>(tid) * N, first_key, K, 0);
        }
        if (bm > bound) push(lds, C::key(bm), static_cast<uint32_t>(i));
      }
    }
  }
  // The columns past the last whole chunk, in the last part.
  const bool has_tail = which == parts - 1;
  const int64_t tail0 = chunks * N;
  float tail = -INFINITY;
  if (has_tail) {                                // (whole wavefronts: the others add nothing)
    if (tail0 + tid < rows.V) tail = Elem<T>::load1(row + (tail0 + tid) * kSize);
    if (tid < kWave) absorb(st, mc, limit, odd, OneColumn{tail}, tail, c, lag);
  }
  move_max(st, fmaxf(tmax, tail), c);
  const Stats total = merge_stats(stat_lds, st, c);
  const int64_t at = r * parts + which;
  const float lse = log_sum(total, c);
  if (tid == 0) {
    if (parts > 1) part.stats[at] = total;
    else write_row<T>(out, r, total, row, rows.V, tokens[r], inv_t, lse);
  }
  if constexpr (TOP) {
    // The chunks that reach the bound of all whole chunks, column by column; the columns that equal a
    // bound, if it is that one; the tail.  (merge_stats synchronised the workgroup: the lists are
    // complete.)
    int count = lds.count;
    const uint32_t key = steps > 0 ? raise_bound<C::kBits>(lds, C::key(tmax), K) : 0u;
    uint32_t apart = kLpThreads;                 // chunks whose equal columns are listed by themselves
    if (count > kListCap) {
      list_again<T>(lds, base, n, col_base, key, K);
      count = lds.count;
      first_key = key;
      apart = static_cast<uint32_t>(n);
    }
    for (int i = tid; i < min(count, kListCap); i += kLpThreads) {
      const Cand e = lds.list[i];
      if (e.key < key) continue;
      C w;
      w.template load<!KEEP>(base, e.col * 16u);
      float z[N];
      w.unpack(z);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t k = C::key(z[j]);
        if (k >= key && !(e.col < apart && k == first_key)) keep(lds, k, col_base + e.col * N + j);
      }
    }
    if (first_key == key && tid < lds.ties) keep(lds, lds.tie[tid].key, lds.tie[tid].col);
    if (has_tail && tail0 + tid < rows.V) keep(lds, C::key(tail), static_cast<uint32_t>(tail0 + tid));
    __syncthreads();
    if (count > kListCap || lds.kept > kKeepCap)
      search_top<T>(lds, row, min(first, chunks) * N, has_tail ? rows.V : last * N, K);
    else
      rank_list(lds, lds.list + kListCap, lds.kept, K, lds.top);
    __syncthreads();
    if (tid < K) {
      const Cand e = lds.top[tid];
      if (parts > 1) {
        part.cand[at * K + tid] = e;
      } else {
        out.top_id[r * K + tid] = e.col;
        out.top_lp[r * K + tid] = column_lp<T>(row, e.col, total, inv_t, lse);
      }
    }
  }
}

// The rows of several parts: lane l of every wavefront holds part l's statistics.  The K best of all
// parts' alternatives are found as in the parts: a bound, the list of what reaches it, ranks.
template <typename T, bool TOP>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_join_kernel(
    const char* __restrict__ logits, const int64_t* __restrict__ tokens, LpRows rows, float c,
    float inv_t, int K, int parts, PartOut part, RowOut out) {
  using C = Chunk<T>;
  __shared__ std::conditional_t<TOP, ListLds, int> lds;
  // Without alternatives a wavefront takes a row.
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t r = TOP ? static_cast<int64_t>(blockIdx.x)
                        : static_cast<int64_t>(blockIdx.x) * kLpWaves + wave;
  if (r >= rows.count) return;
  const char* const row = logits + rows.at(r) * Elem<T>::kBytes;
  Stats st{-INFINITY, 0.f, 0.f};
  if (lane < parts) st = part.stats[r * parts + lane];
  move_max(st, wave_max(st.m), c);
  st.s = wave_sum(st.s);
  st.a = wave_sum(st.a);
  const float lse = log_sum(st, c);
  if (lane == 0 && (!TOP || wave == 0)) write_row<T>(out, r, st, row, rows.V, tokens[r], inv_t, lse);
  if constexpr (TOP) {
    const int tid = threadIdx.x;
    const Cand* const all = part.cand + r * parts * K;
    const int n = parts * K;                       // <= 64 * 32
    if (tid == 0) lds.kept = 0;
    constexpr int kOwn = kMaxParts * kMaxTop / kLpThreads;
    uint32_t best = 0;
    Cand mine[kOwn];
#pragma unroll
    for (int u = 0; u < kOwn; ++u) {
      const int i = u * kLpThreads + tid;
      mine[u] = i < n ? all[i] : Cand{0, kNoCol};
      if (mine[u].col != kNoCol) best = max(best, mine[u].key);
    }
    const uint32_t bound_key = raise_bound<C::kBits>(lds, best, K);
    static_assert(kMaxParts * kMaxTop <= kListCap + kKeepCap, "the list holds every candidate");
#pragma unroll
    for (int u = 0; u < kOwn; ++u)
      if (mine[u].col != kNoCol && mine[u].key >= bound_key)
        lds.list[atomicAdd(&lds.kept, 1)] = mine[u];
    __syncthreads();
    rank_list(lds, lds.list, lds.kept, K, lds.top);
    __syncthreads();
    if (tid < K) {
      const Cand e = lds.top[tid];
      out.top_id[r * K + tid] = e.col;
      out.top_lp[r * K + tid] = column_lp<T>(row, e.col, st, inv_t, lse);
    }
  }
}

// ---- gradient -----------------------------------------------------------------------------------

struct LpGrads {
  const float *row_max, *row_sum, *entropy;
  const float *g_lp, *g_ent, *g_top;   // each nullable
  const int64_t* top_id;
};

// Workgroup (block of chunks, row).  dz = 2^x (k0 + k1 x), x as in the forward and the row's factors k0,
// k1; then the few columns with a gradient of their own are written again by the thread that wrote them.
template <typename T>
__global__ __launch_bounds__(kGradThreads) void token_logprobs_bwd_kernel(
    const char* __restrict__ logits, const int64_t* __restrict__ tokens, LpRows rows, float c,
    float inv_t, int K, int64_t r0, int blocks, LpGrads g, char* __restrict__ dlogits) {
  constexpr int N = Chunk<T>::N;
  constexpr int kSize = Elem<T>::kBytes;
  const int64_t r = r0 + blockIdx.x / static_cast<uint32_t>(blocks);
  const int which = static_cast<int>(blockIdx.x % static_cast<uint32_t>(blocks));
  const char* const row = logits + rows.at(r) * kSize;
  char* const drow = dlogits + r * rows.V * kSize;
  const int tid = threadIdx.x;
  // The columns with a gradient of their own, one a lane in every wavefront: the alternatives' in lanes
  // 0 .. K - 1, the token's in lane 63.
  const int lane = tid & 63;
  const int64_t tok = tokens[r];
  const bool has_tok = g.g_lp != nullptr && tok >= 0 && tok < rows.V;
  int64_t col = -1;
  float g_col = 0.f;
  if (lane == 63 && has_tok) {
    col = tok;
    g_col = g.g_lp[r];
  }
  if (g.g_top != nullptr && lane < K) {
    col = g.top_id[r * K + lane];
    g_col = g.g_top[r * K + lane];
  }
  const float g_ent = g.g_ent != nullptr ? g.g_ent[r] : 0.f;
  const float weight = wave_sum(g_col);
  const bool none = g_ent == 0.f && !__any(g_col != 0.f);
  const float m = g.row_max[r], sum = g.row_sum[r];
  const float inv_s = 1.0f / sum;
  const float lse = logf(sum);
  // -(1/T) p (weight + g_ent (ln p + H)), p = 2^x / S, ln p = x ln 2 - ln S
  const float k1 = none ? 0.f : -inv_t * inv_s * (g_ent * kLn2);
  const float k0 = none ? 0.f : -inv_t * inv_s * (weight + g_ent * (g.entropy[r] - lse));
  const int64_t chunks = rows.V / N;
  const int64_t first = static_cast<int64_t>(which) * (kGradThreads * kGradUnroll) + tid;
  Chunk<T> w[kGradUnroll];
  if (!none) {
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u) {
      const int64_t i = first + u * kGradThreads;
      if (i < chunks) w[u].template load<true>(row + i * 16, 0);
    }
  }
  const float mc = m * c;
  const bool plain = plain_form(mc);
  auto dense = [&](float z) {
    const float x = plain ? __builtin_fmaf(z, c, -mc) : exponent(z, m, mc, c);
    return __builtin_amdgcn_exp2f(x) * __builtin_fmaf(k1, fmaxf(x, kFloor), k0);
  };
#pragma unroll
  for (int u = 0; u < kGradUnroll; ++u) {
    const int64_t i = first + u * kGradThreads;
    if (i >= chunks) continue;
    float z[N];
    if (none) {
#pragma unroll
      for (int j = 0; j < N; ++j) z[j] = 0.f;
    } else {
      w[u].unpack(z);
#pragma unroll
      for (int j = 0; j < N; ++j) z[j] = dense(z[j]);
    }
    Chunk<T>::store(drow + i * 16, z);
  }
  const bool has_tail = which == blocks - 1;
  const int64_t tail = chunks * N + tid;
  if (has_tail && tail < rows.V)
    Elem<T>::store1(drow + tail * kSize,
                    none ? 0.f : dense(Elem<T>::load1(row + tail * kSize)));
  if (none) return;
  // Those of them that lie in this workgroup's columns are written again, each by the thread that wrote
  // it before (its stores to one address stay in order), with the gradients of all its mentions.
  const int64_t at = col / N;
  const bool here = col >= 0 && col < rows.V &&
                    (at < chunks ? at / (kGradThreads * kGradUnroll) == which : has_tail);
  for (uint64_t left = __ballot(here); left != 0; left &= left - 1) {
    const int k = __builtin_ctzll(left);
    const int64_t one =
        static_cast<int64_t>(static_cast<uint32_t>(
            __builtin_amdgcn_readlane(static_cast<int>(col), k)));   // (a column: below 2^31)
    const float add = wave_sum(col == one ? g_col : 0.f);
    const int64_t chunk = one / N;
    const int owner = static_cast<int>(chunk < chunks ? chunk % kGradThreads : one - chunks * N);
    if (owner != tid) continue;
    const float z = Elem<T>::load1(row + one * kSize);
    Elem<T>::store1(drow + one * kSize, dense(z) + add * inv_t);
  }
}

int64_t lp_align(int64_t v) { return (v + 255) / 256 * 256; }

// Parts per row: enough workgroups to fill the chip, each with two steps at least.
int lp_parts(int64_t rows, int64_t V, int32_t dtype, int32_t top_k) {
  const int64_t chunks = V / (dtype == SOUPK_DTYPE_F32 ? 4 : 8);
  const int64_t steps = (chunks + kLpThreads - 1) / kLpThreads;
  const int64_t fill = int64_t{top_k > 0 ? kLpFillTop : kLpFill} * device_cu_count();
  const int64_t want = rows > 0 ? std::max<int64_t>(1, (fill + rows / 2) / rows) : 1;
  const int64_t least = steps * kLpThreads / (int64_t{1} << 27) + 1;   // (32-bit offsets in a part)
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(want, kMaxParts));
  const int64_t per = std::max<int64_t>(2, (steps + parts - 1) / parts);
  return static_cast<int>(std::max<int64_t>(least, (steps + per - 1) / per));
}

bool bad_dtype(int32_t d) {
  return d != SOUPK_DTYPE_F16 && d != SOUPK_DTYPE_BF16 && d != SOUPK_DTYPE_F32;
}

bool bad_lp(int32_t dtype, int64_t rows, int64_t inner, int64_t V, float temperature) {
  return bad_dtype(dtype) || rows < 0 || rows > 0x7fffffff / kMaxParts || inner < 1 || V < 1 ||
         V >= (int64_t{1} << 31) - 16 ||
         !(temperature >= 1e-30f && temperature <= 1e30f);   // (1 / T and log2(e) / T are fp32 numbers)
}

}  // namespace
}  // namespace soupk

using namespace soupk;

extern "C" __attribute__((visibility("default"))) int soupk_token_logprobs_workspace(
    int64_t rows, int64_t V, int32_t top_k, int32_t dtype, int64_t* bytes) {
  if (bad_lp(dtype, rows, 1, V, 1.f) || top_k < 0 || top_k > kMaxTop || bytes == nullptr)
    return kInvalid;
  const int parts = lp_parts(rows, V, dtype, top_k);
  *bytes = parts == 1 ? 0
                      : lp_align(rows * parts * static_cast<int64_t>(sizeof(Stats))) +
                            rows * parts * top_k * static_cast<int64_t>(sizeof(Cand));
  return kOk;
}

extern "C" __attribute__((visibility("default"))) int soupk_token_logprobs_fwd(
    const void* logits, int32_t dtype, const int64_t* tokens, int64_t rows, int64_t inner,
    int64_t stride_outer, int64_t stride_inner, int64_t V, float temperature, int32_t top_k,
    float* logprob, float* entropy, float* row_max, float* row_sum, float* top_lp, int64_t* top_id,
    void* workspace, int64_t workspace_bytes, void* stream) {
  if (bad_lp(dtype, rows, inner, V, temperature)) return kInvalid;
  if (top_k < 0 || top_k > kMaxTop || top_k > V) return kInvalid;
  if (rows == 0) return kOk;
  if (bad_elem_ptr(logits, dtype) || !tokens || !logprob || !entropy ||
      (row_max == nullptr) != (row_sum == nullptr))
    return kInvalid;
  if (top_k > 0 && (!top_lp || !top_id)) return kInvalid;
  int64_t need = 0;
  if (soupk_token_logprobs_workspace(rows, V, top_k, dtype, &need) != kOk) return kInvalid;
  if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) ||
                   workspace_bytes < need))
    return kInvalid;
  const int parts = lp_parts(rows, V, dtype, top_k);
  const float inv_t = 1.0f / temperature;
  const float c = static_cast<float>(1.4426950408889634 / static_cast<double>(temperature));
  const LpRows lr{inner, stride_outer, stride_inner, V, rows};
  const PartOut po{static_cast<Stats*>(workspace),
                   reinterpret_cast<Cand*>(static_cast<char*>(workspace) +
                                           lp_align(rows * parts *
                                                    static_cast<int64_t>(sizeof(Stats))))};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto tag) -> int {
    using T = typename decltype(tag)::type;
    const int64_t chunks = V / Chunk<T>::N;
    const int64_t part_chunks = (chunks + parts - 1) / parts;
    const RowOut ro{logprob, entropy, row_max, row_sum, top_lp, top_id};
    auto run = [&](auto kernel) {
      const int64_t most = kMaxGrid / parts;         // rows of one launch
      for (int64_t r0 = 0; r0 < rows; r0 += most) {
        const int64_t n = std::min(most, rows - r0);
        const int rc = launch_kernel(kernel, dim3(static_cast<unsigned>(n * parts)), dim3(kLpThreads),
                                     s, static_cast<const char*>(logits), tokens, lr, c, inv_t,
                                     static_cast<int>(top_k), parts, part_chunks, r0, po, ro);
        if (rc != kOk) return rc;
      }
      return static_cast<int>(kOk);
    };
    const bool keep = row_max != nullptr;       // (asked for by a backward)
    const int rc = top_k > 0 ? keep ? run(token_logprobs_kernel<T, true, true>)
                                    : run(token_logprobs_kernel<T, true, false>)
                   : keep    ? run(token_logprobs_kernel<T, false, true>)
                             : run(token_logprobs_kernel<T, false, false>);
    if (rc != kOk || parts == 1) return rc;
    auto join = [&](auto kernel, int64_t blocks) {
      return launch_kernel(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kLpThreads), s,
                           static_cast<const char*>(logits), tokens, lr, c, inv_t,
                           static_cast<int>(top_k), parts, po, ro);
    };
    return top_k > 0 ? join(token_logprobs_join_kernel<T, true>, rows)
                     : join(token_logprobs_join_kernel<T, false>, (rows + kLpWaves - 1) / kLpWaves);
  });
}

extern "C" __attribute__((visibility("default"))) int soupk_token_logprobs_bwd(
    const void* logits, int32_t dtype, const int64_t* tokens, int64_t rows, int64_t inner,
    int64_t stride_outer, int64_t stride_inner, int64_t V, float temperature, int32_t top_k,
    const float* row_max, const float* row_sum, const float* entropy, const int64_t* top_id,
    const float* g_lp, const float* g_ent, const float* g_top, void* dlogits, void* stream) {
  if (bad_lp(dtype, rows, inner, V, temperature)) return kInvalid;
  if (top_k < 0 || top_k > kMaxTop || top_k > V) return kInvalid;
  if (rows == 0) return kOk;
  if (bad_elem_ptr(logits, dtype) || bad_elem_ptr(dlogits, dtype) || !tokens || !row_max ||
      !row_sum || !entropy)
    return kInvalid;
  if (g_top != nullptr && (top_k == 0 || !top_id)) return kInvalid;
  const float inv_t = 1.0f / temperature;
  const float c = static_cast<float>(1.4426950408889634 / static_cast<double>(temperature));
  const LpRows lr{inner, stride_outer, stride_inner, V, rows};
  return with_type(dtype, [&](auto tag) -> int {
    using T = typename decltype(tag)::type;
    constexpr int64_t kPer = kGradThreads * kGradUnroll;
    const int64_t blocks = std::max<int64_t>(1, (V / Chunk<T>::N + kPer - 1) / kPer);
    const int64_t most = std::max<int64_t>(1, kMaxGrid / blocks);    // rows of one launch
    for (int64_t r0 = 0; r0 < rows; r0 += most) {
      const int64_t n = std::min(most, rows - r0);
      const int rc = launch_kernel(
          token_logprobs_bwd_kernel<T>, dim3(static_cast<unsigned>(n * blocks)), dim3(kGradThreads),
          static_cast<hipStream_t>(stream), static_cast<const char*>(logits), tokens, lr, c, inv_t,
          static_cast<int>(top_k), r0, static_cast<int>(blocks),
          LpGrads{row_max, row_sum, entropy, g_lp, g_ent, g_top, top_id},
          static_cast<char*>(dlogits));
      if (rc != kOk) return rc;
    }
    return kOk;
  });
}
