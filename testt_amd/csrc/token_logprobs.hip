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
// among the K, and goes into a short list in LDS.  The bound is raised after 1, 2, 8, 32, ... steps,
// so the list stays at some ten times K entries whatever the row's length.  Columns of the first step are
// listed by the bound found from it, equal ones only as far as they can count (by their order).  At the
// end the list is ranked.  A row that rises so steadily that the list overflows (no such row comes from
// a model) is ranked by K searches over the row instead.
//
// Few rows are cut into parts, whose statistics and alternatives a second launch joins.

#include <algorithm>
#include <type_traits>

#include "elem.hpp"

namespace soupk {
namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / kWave;
constexpr int kLpUnroll = 4;          // chunk loads in flight per thread
constexpr int kMaxTop = 32;
constexpr int kListCap = 1024;        // candidates of a part
constexpr int kMaxParts = 64;
constexpr int64_t kIgnored = -100;
constexpr float kFloor = -200.f;      // below 2^kFloor an exponential is zero in fp32

// Rows of the logits: row r is (r / inner, r % inner) with its two strides (elements).
struct LpRows {
  int64_t inner, stride_outer, stride_inner, V;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    const int64_t o = r / inner;
    return o * stride_outer + (r - o * inner) * stride_inner;
  }
};

// A 16-byte chunk as floats: 8 half-size or 4 fp32 columns.
template <typename T>
struct Chunk {
  static constexpr int N = 16 / Elem<T>::kBytes;
  u32x4 w;
  __device__ __forceinline__ void load(const char* p) {
    w = ld<true>(reinterpret_cast<const u32x4_a2*>(p));
  }
  __device__ __forceinline__ void unpack(float* v) const {
    if constexpr (std::is_same_v<T, float>) {
      const f32x4 f = __builtin_bit_cast(f32x4, w);
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
      Elem<T>::unpack8(typename Elem<T>::Raw8{w}, v);
    }
  }
  static __device__ __forceinline__ void store(char* p, const float* v) {
    if constexpr (std::is_same_v<T, float>)
      st<true>(reinterpret_cast<f32x4_a4*>(p), static_cast<f32x4_a4>(f32x4{v[0], v[1], v[2], v[3]}));
    else
      Elem<T>::template store8<true>(p, v);
  }
};

// Running statistics: the maximum, S = sum 2^x and A = sum 2^x x with x = (z - m) * c, c = log2(e) / T.
struct Stats {
  float m, s, a;
};

__device__ __forceinline__ float shifted(float z, float m, float c) {
  return (z - (m == -INFINITY ? 0.f : m)) * c;      // (a part of -inf alone: 2^-inf = 0)
}

// The statistics relative to another maximum m >= st.m.
__device__ __forceinline__ void move_max(Stats& st, float m, float c) {
  if (st.m == m) return;
  const float x = fmaxf((st.m - m) * c, kFloor);    // (st.m = -inf: s and a are 0)
  const float f = st.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x);
  st.a = f * (st.a + x * st.s);
  st.s = f * st.s;
  st.m = m;
}

template <int N>
__device__ __forceinline__ void absorb(Stats& st, const float* z, float bm, float c) {
  if (bm > st.m) move_max(st, bm, c);
  const float m = st.m == -INFINITY ? 0.f : st.m;
  float e[N], x[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    x[j] = (z[j] - m) * c;
    e[j] = __builtin_amdgcn_exp2f(x[j]);
  }
  float s = 0.f, a = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    s = s + e[j];
    a = __builtin_fmaf(e[j], fmaxf(x[j], kFloor), a);
  }
  st.s = st.s + s;
  st.a = st.a + a;
}

// fp32 bits in an order that integers compare; NaN as -inf, -0 as 0.
__device__ __forceinline__ uint32_t sort_bits(float z) {
  if (z != z) z = -INFINITY;
  if (z == 0.f) z = 0.f;
  const uint32_t b = __builtin_bit_cast(uint32_t, z);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unsort_bits(uint32_t k) {
  return __builtin_bit_cast(float, (k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

struct Cand {
  uint32_t key;   // sort_bits of the value
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
  Cand list[kListCap];
  Cand keep[kListCap];
  uint32_t group_max[64];
  int count, kept;
  int wave_n[kLpWaves];
  Cand best[kLpWaves];
};

// The K-th largest of the 64 groups' maxima (a group: 4 neighbouring threads); every thread of the
// workgroup calls it and gets it.
__device__ __forceinline__ uint32_t raise_bound(ListLds& s, float tmax, int K) {
  const int lane = threadIdx.x & 63;
  uint32_t k = sort_bits(tmax);
  k = max(k, static_cast<uint32_t>(dpp_i<kDppQuad1032>(static_cast<int>(k))));
  k = max(k, static_cast<uint32_t>(dpp_i<kDppQuad2301>(static_cast<int>(k))));
  __syncthreads();                               // (group_max of the last call has been read)
  if ((threadIdx.x & 3) == 0) s.group_max[threadIdx.x >> 2] = k;
  __syncthreads();
  const uint32_t mine = s.group_max[lane];
  uint32_t bound = 0;
#pragma unroll
  for (int b = 31; b >= 0; --b) {
    const uint32_t cand = bound | (1u << b);
    if (__popcll(__ballot(mine >= cand)) >= K) bound = cand;
  }
  return bound;
}

__device__ __forceinline__ void push(ListLds& s, uint32_t key, uint32_t col) {
  const int at = atomicAdd(&s.count, 1);
  if (at < kListCap) s.list[at] = Cand{key, col};
}

// Writes the K best of n candidates in order (entries past the last one have column kNoCol); every
// thread of the workgroup calls it.
__device__ __forceinline__ void rank_list(const Cand* list, int n, int K, Cand* out) {
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
__device__ void search_top(ListLds& s, const char* row, int64_t col0, int64_t col1, int K,
                           Cand* out) {
  Cand last{0xffffffffu, 0};
  bool any = true;
  for (int k = 0; k < K; ++k) {
    Cand best{0, kNoCol};
    if (any)
      for (int64_t i = col0 + threadIdx.x; i < col1; i += kLpThreads) {
        const Cand c{sort_bits(Elem<T>::load1(row + i * Elem<T>::kBytes)),
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
    if (threadIdx.x == 0) out[k] = best;
    any = best.col != kNoCol;
    last = best;
    __syncthreads();
  }
}

// Statistics of the workgroup, in every thread of its first wavefront.
__device__ __forceinline__ Stats merge_stats(Stats* lds, Stats st, float c) {
  auto across = [&](float v, auto f) {
    for (int d = 32; d > 0; d >>= 1) v = f(v, __shfl_xor(v, d));
    return v;
  };
  const float m = across(st.m, [](float a, float b) { return fmaxf(a, b); });
  move_max(st, m, c);
  st.s = across(st.s, [](float a, float b) { return a + b; });
  st.a = across(st.a, [](float a, float b) { return a + b; });
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

// The numbers of a row from its statistics (one thread).
template <typename T>
__device__ __forceinline__ float write_row(const RowOut& o, int64_t r, const Stats& st,
                                           const char* row, int64_t V, int64_t tok, float inv_t) {
  // (a row without a finite maximum: NaN, as the formula gives)
  const float lse = st.m > -INFINITY ? logf(st.s) : NAN;
  o.entropy[r] = lse - kLn2 * (st.a / st.s);
  float lp = NAN;
  if (tok == kIgnored) lp = 0.f;
  else if (tok >= 0 && tok < V)
    lp = (Elem<T>::load1(row + tok * Elem<T>::kBytes) - st.m) * inv_t - lse;
  o.logprob[r] = lp;
  if (o.row_max != nullptr) {
    o.row_max[r] = st.m;
    o.row_sum[r] = st.s;
  }
  return lse;
}

template <typename T, bool TOP>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_kernel(
    const char* __restrict__ logits, const int64_t* __restrict__ tokens, LpRows rows, float c,
    float inv_t, int K, int parts, int64_t part_chunks, PartOut part, RowOut out) {
  constexpr int N = Chunk<T>::N;
  constexpr int kSize = Elem<T>::kBytes;
  __shared__ Stats stat_lds[kLpWaves];
  __shared__ std::conditional_t<TOP, ListLds, int> lds;
  const int64_t r = blockIdx.x / static_cast<uint32_t>(parts);
  const int which = static_cast<int>(blockIdx.x % static_cast<uint32_t>(parts));
  const char* const row = logits + rows.at(r) * kSize;
  const int64_t chunks = rows.V / N;
  const int64_t first = which * part_chunks;
  const int64_t last = min(chunks, first + part_chunks);
  const int tid = threadIdx.x;
  Stats st{-INFINITY, 0.f, 0.f};
  float tmax = -INFINITY;        // this thread's largest value so far (never NaN)
  uint32_t bound_key = 0;
  float bound = -INFINITY;
  if constexpr (TOP) {
    if (tid == 0) lds.count = lds.kept = 0;
    __syncthreads();
  }
  const char* const p0 = row + (first + tid) * 16;
  const int64_t n = last - first - tid;          // chunks of this thread: every 256th
  const int64_t steps = (last - first + kLpThreads - 1) / kLpThreads;
  int64_t next_raise = 2;
  for (int64_t step = 0; step < steps; step += kLpUnroll) {
    Chunk<T> w[kLpUnroll];
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      // (past the part's end: its first chunk, unused, so that no load waits for a branch)
      const int64_t i = (step + u) * kLpThreads;
      w[u].load(i < n ? p0 + i * 16 : row + first * 16);
    }
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      if constexpr (TOP) {
        if (step + u == next_raise && step + u < steps) {
          next_raise *= 4;
          bound_key = raise_bound(lds, tmax, K);
          bound = unsort_bits(bound_key);
        }
      }
      const int64_t i = (step + u) * kLpThreads;
      const bool on = i < n;
      float z[N];
      if (on) {
        w[u].unpack(z);
        float bm = z[0];
#pragma unroll
        for (int j = 1; j < N; ++j) bm = fmaxf(bm, z[j]);
        absorb<N>(st, z, bm, c);
        if constexpr (TOP) {
          tmax = fmaxf(tmax, bm);
          if (step + u > 0 && bm > bound) {
            const uint32_t col = static_cast<uint32_t>((first + tid + i) * N);
#pragma unroll
            for (int j = 0; j < N; ++j)
              if (z[j] > bound) push(lds, sort_bits(z[j]), col + j);
          }
        }
      }
      if constexpr (TOP) {
        if (step + u == 0) {
          // The first step's columns against the bound that they give: those above it, and as many of
          // the equal ones, from the left, as the K can still take.
          bound_key = raise_bound(lds, tmax, K);
          uint32_t key[N];
          int above = 0, equal = 0;
          if (on) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
              key[j] = sort_bits(z[j]);
              above += key[j] > bound_key ? 1 : 0;
              equal += key[j] == bound_key ? 1 : 0;
            }
          }
          // equal columns left of this thread's, by a scan over the workgroup
          int upto = equal;
          for (int d = 1; d < kWave; d <<= 1) {
            const int v = __shfl_up(upto, d);
            if ((tid & 63) >= d) upto += v;
          }
          if ((tid & 63) == 63) lds.wave_n[tid >> 6] = upto;
          __syncthreads();
          int left = upto - equal;
          for (int k = 0; k < (tid >> 6); ++k) left += lds.wave_n[k];
          if (on && (above > 0 || (equal > 0 && left < K))) {
            const uint32_t col = static_cast<uint32_t>((first + tid) * N);
#pragma unroll
            for (int j = 0; j < N; ++j) {
              if (key[j] > bound_key) push(lds, key[j], col + j);
              if (key[j] == bound_key) {
                if (left < K) push(lds, key[j], col + j);
                ++left;
              }
            }
          }
          bound = unsort_bits(bound_key);
        }
      }
    }
  }
  // The columns past the last whole chunk, in the last part.
  const bool has_tail = last == chunks && which == parts - 1;
  const int64_t tail0 = chunks * N;
  if (has_tail && tail0 + tid < rows.V) {
    const float z = Elem<T>::load1(row + (tail0 + tid) * kSize);
    absorb<1>(st, &z, z, c);
    if constexpr (TOP) push(lds, sort_bits(z), static_cast<uint32_t>(tail0 + tid));
  }
  const Stats total = merge_stats(stat_lds, st, c);
  const int64_t at = blockIdx.x;
  float lse = 0.f;
  if (parts > 1) {
    if (tid == 0) part.stats[at] = total;
  } else if (tid < 64) {
    lse = total.m > -INFINITY ? logf(total.s) : NAN;
    if (tid == 0) write_row<T>(out, r, total, row, rows.V, tokens[r], inv_t);
  }
  if constexpr (TOP) {
    // (merge_stats synchronised the workgroup: the list is complete)
    __shared__ Cand top[kMaxTop];
    const int count = lds.count;
    if (count > kListCap) {
      search_top<T>(lds, row, first * N, has_tail ? rows.V : last * N, K, top);
    } else {
      bound_key = raise_bound(lds, tmax, K);     // of all whole chunks: what is below it is out
      for (int i = tid; i < count; i += kLpThreads)
        if (lds.list[i].key >= bound_key) lds.keep[atomicAdd(&lds.kept, 1)] = lds.list[i];
      __syncthreads();
      rank_list(lds.keep, lds.kept, K, top);
    }
    __syncthreads();
    if (tid < K) {
      const Cand e = top[tid];
      if (parts > 1) {
        part.cand[at * K + tid] = e;
      } else {
        const float z = Elem<T>::load1(row + static_cast<int64_t>(e.col) * kSize);
        out.top_id[r * K + tid] = e.col;
        out.top_lp[r * K + tid] = (z - total.m) * inv_t - lse;
      }
    }
  }
}

// One wavefront per row: lane l holds part l.  The alternatives are merged by K rounds over the heads
// of the parts' lists.
template <typename T>
__global__ __launch_bounds__(kWave) void token_logprobs_join_kernel(
    const char* __restrict__ logits, const int64_t* __restrict__ tokens, LpRows rows, float c,
    float inv_t, int K, int parts, PartOut part, RowOut out) {
  const int64_t r = blockIdx.x;
  const char* const row = logits + rows.at(r) * Elem<T>::kBytes;
  const int lane = threadIdx.x;
  Stats st{-INFINITY, 0.f, 0.f};
  if (lane < parts) st = part.stats[r * parts + lane];
  float m = st.m;
  for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  move_max(st, m, c);
  for (int d = 32; d > 0; d >>= 1) {
    st.s = st.s + __shfl_xor(st.s, d);
    st.a = st.a + __shfl_xor(st.a, d);
  }
  const float lse = st.m > -INFINITY ? logf(st.s) : NAN;
  if (lane == 0) write_row<T>(out, r, st, row, rows.V, tokens[r], inv_t);
  if (K == 0) return;
  const Cand* const mine = part.cand + (r * parts + lane) * K;
  int at = 0;
  Cand head = lane < parts ? mine[0] : Cand{0, kNoCol};
  for (int k = 0; k < K; ++k) {
    Cand best = head;
    for (int d = 32; d > 0; d >>= 1) {
      const Cand o{__shfl_xor(best.key, d), __shfl_xor(best.col, d)};
      if (ahead(o, best)) best = o;
    }
    if (head.col == best.col && head.col != kNoCol) {
      const float z = Elem<T>::load1(row + static_cast<int64_t>(best.col) * Elem<T>::kBytes);
      out.top_id[r * K + k] = best.col;
      out.top_lp[r * K + k] = (z - m) * inv_t - lse;
      ++at;
      head = at < K ? mine[at] : Cand{0, kNoCol};
    }
  }
}

// ---- gradient -----------------------------------------------------------------------------------

struct LpGrads {
  const float *row_max, *row_sum, *entropy;
  const float *g_lp, *g_ent, *g_top;   // each nullable
  const int64_t* top_id;
};

// Workgroup (block of chunks, row).  dz = 2^x (k0 + k1 x) with x = (z - m) c and the row's factors k0,
// k1; then the few columns with a gradient of their own are written again by the thread that wrote them.
template <typename T>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_bwd_kernel(
    const char* __restrict__ logits, const int64_t* __restrict__ tokens, LpRows rows, float c,
    float inv_t, int K, int64_t r0, int blocks, LpGrads g, char* __restrict__ dlogits) {
  constexpr int N = Chunk<T>::N;
  constexpr int kSize = Elem<T>::kBytes;
  const int64_t r = r0 + blockIdx.x / static_cast<uint32_t>(blocks);
  const int which = static_cast<int>(blockIdx.x % static_cast<uint32_t>(blocks));
  const char* const row = logits + rows.at(r) * kSize;
  char* const drow = dlogits + r * rows.V * kSize;
  const int tid = threadIdx.x;
  const int64_t tok = tokens[r];
  const bool has_tok = g.g_lp != nullptr && tok >= 0 && tok < rows.V;
  const float g_tok = has_tok ? g.g_lp[r] : 0.f;
  const float g_ent = g.g_ent != nullptr ? g.g_ent[r] : 0.f;
  float weight = g_tok;
  bool none = g_tok == 0.f && g_ent == 0.f;
  if (g.g_top != nullptr)
    for (int k = 0; k < K; ++k) {
      const float v = g.g_top[r * K + k];
      weight = weight + v;
      none = none && v == 0.f;
    }
  const float m = g.row_max[r], sum = g.row_sum[r];
  const float inv_s = 1.0f / sum;
  const float lse = logf(sum);
  // -(1/T) p (weight + g_ent (ln p + H)), p = 2^x / S, ln p = x ln 2 - ln S
  const float k1 = none ? 0.f : -inv_t * inv_s * (g_ent * kLn2);
  const float k0 = none ? 0.f : -inv_t * inv_s * (weight + g_ent * (g.entropy[r] - lse));
  const int64_t chunks = rows.V / N;
  const int64_t first = static_cast<int64_t>(which) * (kLpThreads * kLpUnroll) + tid;
  Chunk<T> w[kLpUnroll];
  if (!none) {
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      const int64_t i = first + u * kLpThreads;
      if (i < chunks) w[u].load(row + i * 16);
    }
  }
  auto dense = [&](float z) {
    const float x = (z - m) * c;
    return __builtin_amdgcn_exp2f(x) * __builtin_fmaf(k1, fmaxf(x, kFloor), k0);
  };
#pragma unroll
  for (int u = 0; u < kLpUnroll; ++u) {
    const int64_t i = first + u * kLpThreads;
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
  // The token's column and the alternatives': -1 stands for the token.
  const int tops = g.g_top != nullptr ? K : 0;
  for (int k = has_tok ? -1 : 0; k < tops; ++k) {
    const int64_t col = k < 0 ? tok : g.top_id[r * K + k];
    if (col < 0 || col >= rows.V) continue;
    const int64_t i = col / N;
    const bool own = i < chunks ? i % kLpThreads == tid &&
                                      i / (kLpThreads * kLpUnroll) == which
                                : has_tail && col - chunks * N == tid;
    if (!own) continue;
    float add = 0.f;
    for (int q = has_tok ? -1 : 0; q < tops; ++q)
      if ((q < 0 ? tok : g.top_id[r * K + q]) == col)
        add = add + (q < 0 ? g_tok : g.g_top[r * K + q]);
    const float z = Elem<T>::load1(row + col * kSize);
    Elem<T>::store1(drow + col * kSize, dense(z) + add * inv_t);
  }
}

int64_t lp_align(int64_t v) { return (v + 255) / 256 * 256; }

// Parts per row: enough workgroups to fill the chip, each with at least kMinSteps steps.
int lp_parts(int64_t rows, int64_t V, int32_t dtype) {
  const int64_t chunks = V / (dtype == SOUPK_DTYPE_F32 ? 4 : 8);
  const int64_t steps = (chunks + kLpThreads - 1) / kLpThreads;
  const int64_t want = rows > 0 ? (int64_t{4} * device_cu_count() + rows - 1) / rows : 1;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, steps / 2, kMaxParts})));
}

bool bad_dtype(int32_t d) {
  return d != SOUPK_DTYPE_F16 && d != SOUPK_DTYPE_BF16 && d != SOUPK_DTYPE_F32;
}

bool bad_lp(int32_t dtype, int64_t rows, int64_t inner, int64_t V, float temperature) {
  return bad_dtype(dtype) || rows < 0 || rows > 0x7fffffff / kMaxParts || inner < 1 || V < 1 ||
         V >= (int64_t{1} << 31) - 16 || !(temperature > 0.f) || temperature > 3e38f;
}

}  // namespace
}  // namespace soupk

using namespace soupk;

extern "C" __attribute__((visibility("default"))) int soupk_token_logprobs_workspace(
    int64_t rows, int64_t V, int32_t top_k, int32_t dtype, int64_t* bytes) {
  if (bad_lp(dtype, rows, 1, V, 1.f) || top_k < 0 || top_k > kMaxTop || bytes == nullptr)
    return kInvalid;
  const int parts = lp_parts(rows, V, dtype);
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
  const int parts = lp_parts(rows, V, dtype);
  const float inv_t = 1.0f / temperature;
  const float c = static_cast<float>(1.4426950408889634 / static_cast<double>(temperature));
  const LpRows lr{inner, stride_outer, stride_inner, V};
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
      return launch_kernel(kernel, dim3(static_cast<unsigned>(rows * parts)), dim3(kLpThreads), s,
                           static_cast<const char*>(logits), tokens, lr, c, inv_t,
                           static_cast<int>(top_k), parts, part_chunks, po, ro);
    };
    int rc = top_k > 0 ? run(token_logprobs_kernel<T, true>)
                       : run(token_logprobs_kernel<T, false>);
    if (rc != kOk || parts == 1) return rc;
    return launch_kernel(token_logprobs_join_kernel<T>, dim3(static_cast<unsigned>(rows)),
                         dim3(kWave), s, static_cast<const char*>(logits), tokens, lr, c, inv_t,
                         static_cast<int>(top_k), parts, po, ro);
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
  const LpRows lr{inner, stride_outer, stride_inner, V};
  return with_type(dtype, [&](auto tag) -> int {
    using T = typename decltype(tag)::type;
    constexpr int64_t kPer = kLpThreads * kLpUnroll;
    const int64_t blocks = std::max<int64_t>(1, (V / Chunk<T>::N + kPer - 1) / kPer);
    const int64_t most = 0x7fffffff / blocks;        // rows of one launch
    for (int64_t r0 = 0; r0 < rows; r0 += most) {
      const int64_t n = std::min(most, rows - r0);
      const int rc = launch_kernel(
          token_logprobs_bwd_kernel<T>, dim3(static_cast<unsigned>(n * blocks)), dim3(kLpThreads),
          static_cast<hipStream_t>(stream), static_cast<const char*>(logits), tokens, lr, c, inv_t,
          static_cast<int>(top_k), r0, static_cast<int>(blocks),
          LpGrads{row_max, row_sum, entropy, g_lp, g_ent, g_top, top_id},
          static_cast<char*>(dlogits));
      if (rc != kOk) return rc;
    }
    return kOk;
  });
}
