// Embedding lookup with a scale, and the gradient of the table.
//
// Forward:  out[i] = table[ids[i]] * scale, in fp32, rounded once to the output's type; an id outside
// [0, V) gives a row of zeros.  Bound by the rows it copies.
//
// Gradient:  dtable[v] = scale * sum of dout[i] over the tokens i with ids[i] = v, zero for the rows
// that no token names (nor for padding_idx).  The tokens are sorted by id, stably, so each row's sum
// runs over its tokens in their order, in fp32, and is rounded once to the table's type: no atomics
// on values, the same bits every time.  Three steps:
//
//   sort    least-significant-digit radix sort of (id, token) by 9-bit digits, ranks from wavefront
//           ballots.  Up to kOneBlock tokens are sorted by one workgroup in one launch; more tokens
//           by up to kMaxBlocks workgroups, a histogram and a scatter launch per digit.  The last pass
//           also notes, per id, the sorted place of one of its tokens.
//   write   the sorted tokens are cut into runs.  A workgroup adds the rows of its run, in order, and
//           writes a table row for each id that lies within the run; an id that continues past an end
//           of the run leaves a partial fp32 row instead.  All other workgroups write zeros, 16 bytes
//           a thread, to the rows that no token names.
//   join    the partial rows of an id that spans runs are added in run order and written.
//
// The whole table gradient has to be written once (467 MB of fp16 at 151936 x 1536), which is by far
// the largest part of the traffic.  Whether a row is named needs no cleared flags: the noted place is
// looked up, whatever the memory holds, and counts only if the sorted id there is the row.  The sort's
// launches, which leave the chip idle, carry zeros for the first rows of the table.
// Zeros go out as one 16-byte store per thread: 467 MB took 70 us that way on MI355X, 84 us with four
// stores a thread, 95 - 115 us from a grid of resident workgroups.

#include <algorithm>
#include <type_traits>

#include "elem.hpp"
#include "fastdiv.hpp"

namespace soupk {
namespace {

constexpr int kEmbThreads = 256;

// A thread takes 16 bytes of the result: a wavefront's store fills whole lines.
template <typename Out>
constexpr int lookup_cols() {
  return 16 / Elem<Out>::kBytes;
}

template <typename In, typename Out>
__global__ __launch_bounds__(kEmbThreads) void embedding_fwd_kernel(
    const char* __restrict__ table, const int64_t* __restrict__ ids, char* __restrict__ out,
    float scale, int64_t V, int64_t H, uint32_t items, int64_t row0, FastDiv per_row) {
  constexpr int N = lookup_cols<Out>();
  const uint32_t i = blockIdx.x * kEmbThreads + threadIdx.x;
  if (i >= items) return;
  const uint32_t r = per_row.div(i);
  const int64_t col = static_cast<int64_t>(i - r * per_row.d) * N;
  const int64_t row = row0 + r;
  const int n = static_cast<int>(min(int64_t{N}, H - col));
  const int64_t id = ids[row];
  const bool known = id >= 0 && id < V;
  const char* src = table + ((known ? id : 0) * H + col) * Elem<In>::kBytes;
  char* dst = out + (row * H + col) * Elem<Out>::kBytes;
  float v[N];
  if (n == N) {
    load_n<In, N, false>(src, v);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = known ? v[j] * scale : 0.f;
    store_n<Out, N, true>(dst, v);
  } else {
    for (int j = 0; j < n; ++j)
      Elem<Out>::store1(dst + j * Elem<Out>::kBytes,
                        known ? Elem<In>::load1(src + j * Elem<In>::kBytes) * scale : 0.f);
  }
}

// ---- sort ---------------------------------------------------------------------------------------

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kMaxBlocks = 64;
constexpr int64_t kOneBlock = 4096;    // tokens that one workgroup sorts alone
// Bytes of zeros that a launch of the sort carries: what the chip writes in its time (one workgroup's
// sort about 11 us, a histogram or scatter 9).  467 MB at 888 tokens 88 us without, 84 with 48 MB, 82
// with 64; at 32768 tokens 138 without, 129 with 32 MB each, 127 with 48, 132 with 80.
constexpr int64_t hidden_bytes(bool small) { return int64_t{small ? 64 : 48} << 20; }

// Sorted positions that one workgroup adds: few when there are few tokens, so that the chip is filled.
__host__ __device__ constexpr int run_length(int64_t M) { return M <= kOneBlock ? 8 : 32; }

struct Zeros {         // 16-byte words of the table gradient, cleared by extra workgroups
  char* base;
  int64_t count;
};

__device__ __forceinline__ void write_zeros(const Zeros& z, int64_t block) {
  const int64_t i = block * kSortThreads + threadIdx.x;
  if (i < z.count) st16<true>(z.base + 16 * i, u32x4{0u, 0u, 0u, 0u});
}

// The id a token sorts by: V (behind every row) for an id that gets no gradient.
__device__ __forceinline__ uint32_t sort_key(int64_t id, int64_t V, int64_t padding) {
  return static_cast<uint32_t>(id >= 0 && id < V && id != padding ? id : V);
}

struct SortLds {
  uint32_t count[kSortWaves][kDigits];
  uint32_t base[kDigits];
  uint32_t wave_sum[kSortWaves];
};

// Exclusive prefix sum of one value per thread of the first kDigits threads, into s.base; every
// thread of the workgroup calls it.
__device__ __forceinline__ void scan_digits(SortLds& s, uint32_t total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t v = threadIdx.x < kDigits ? total : 0u;
  const uint32_t own = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t up = __shfl_up(v, d);
    if (lane >= d) v += up;
  }
  if (lane == 63) s.wave_sum[w] = v;
  __syncthreads();
  uint32_t before = 0;
  for (int k = 0; k < w; ++k) before += s.wave_sum[k];
  if (threadIdx.x < kDigits) s.base[threadIdx.x] += before + v - own;
  __syncthreads();
}

// Moves the tokens [t0, t1) to their places by the digit at `shift`; s.base holds, per digit, the
// place of the workgroup's first token of it.  s.count is clear.  store(place, key, token) is called
// once per token.
template <typename Load, typename Store>
__device__ __forceinline__ void scatter_tokens(SortLds& s, int64_t t0, int64_t t1, int shift,
                                               const Load& load, const Store& store) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int64_t t = t0; t < t1; t += kSortThreads) {
    const int64_t i = t + threadIdx.x;
    const bool on = i < t1;
    uint32_t key = 0, tok = 0;
    if (on) load(i, key, tok);
    const uint32_t digit = (key >> shift) & (kDigits - 1);
    uint64_t same = __ballot(on);
#pragma unroll
    for (int b = 0; b < kDigitBits; ++b) {
      const uint64_t m = __ballot((digit >> b) & 1u);
      same &= (digit >> b) & 1u ? m : ~m;
    }
    const uint32_t rank = __popcll(same & ((uint64_t{1} << lane) - 1));
    const bool leads = on && rank == 0;
    if (leads) s.count[w][digit] = __popcll(same);
    __syncthreads();
    if (threadIdx.x < kDigits) {
      uint32_t at = s.base[threadIdx.x];
#pragma unroll
      for (int k = 0; k < kSortWaves; ++k) {
        const uint32_t n = s.count[k][threadIdx.x];
        s.count[k][threadIdx.x] = at;
        at += n;
      }
      s.base[threadIdx.x] = at;
    }
    __syncthreads();
    if (on) store(s.count[w][digit] + rank, key, tok);
    if (t + kSortThreads >= t1) break;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortWaves * kDigits / kSortThreads; ++k)
      (&s.count[0][0])[k * kSortThreads + threadIdx.x] = 0;
    __syncthreads();
  }
}

__device__ __forceinline__ void clear_counts(SortLds& s) {
#pragma unroll
  for (int k = 0; k < kSortWaves * kDigits / kSortThreads; ++k)
    (&s.count[0][0])[k * kSortThreads + threadIdx.x] = 0;
  if (threadIdx.x < kDigits) s.base[threadIdx.x] = 0;
  __syncthreads();
}

// Up to kOneBlock tokens: all passes in one workgroup; the others clear the table gradient.  The
// sorted pairs end in key[0] / tok[0] for an even number of passes, else in key[1] / tok[1].
__global__ __launch_bounds__(kSortThreads) void embedding_sort_small_kernel(
    const int64_t* __restrict__ ids, int64_t M, int64_t V, int64_t padding, int passes,
    uint32_t* key0, uint32_t* tok0, uint32_t* key1, uint32_t* tok1, uint32_t* place, Zeros z) {
  if (blockIdx.x > 0) {
    write_zeros(z, blockIdx.x - 1);
    return;
  }
  __shared__ SortLds s;
  for (int p = 0; p < passes; ++p) {
    const int shift = p * kDigitBits;
    uint32_t *ik = p & 1 ? key1 : key0, *it = p & 1 ? tok1 : tok0;
    uint32_t *ok = p & 1 ? key0 : key1, *ot = p & 1 ? tok0 : tok1;
    auto load = [&](int64_t i, uint32_t& k, uint32_t& t) {
      if (p == 0) {
        k = sort_key(ids[i], V, padding);
        t = static_cast<uint32_t>(i);
      } else {
        k = ik[i];
        t = it[i];
      }
    };
    clear_counts(s);
    for (int64_t i = threadIdx.x; i < M; i += kSortThreads) {
      uint32_t k, t;
      load(i, k, t);
      atomicAdd(&s.count[0][(k >> shift) & (kDigits - 1)], 1u);
    }
    __syncthreads();
    const uint32_t total = threadIdx.x < kDigits ? s.count[0][threadIdx.x] : 0u;
    __syncthreads();
    if (threadIdx.x < kDigits) s.count[0][threadIdx.x] = 0;
    scan_digits(s, total);
    const bool last = p == passes - 1;
    scatter_tokens(s, 0, M, shift, load, [&](uint32_t to, uint32_t key, uint32_t tok) {
      ok[to] = key;
      ot[to] = tok;
      // (any token's place will do: of an id's several writers any may win)
      if (last && key < static_cast<uint32_t>(V)) place[key] = to;
    });
    __threadfence_block();
    __syncthreads();
  }
}

// More tokens: workgroup b counts the digits of its stretch into hist[digit][b] ...
__global__ __launch_bounds__(kSortThreads) void embedding_hist_kernel(
    const int64_t* __restrict__ ids, const uint32_t* __restrict__ in_key, int64_t M, int64_t V,
    int64_t padding, int shift, int blocks, int64_t per, uint32_t* __restrict__ hist, Zeros z) {
  if (static_cast<int>(blockIdx.x) >= blocks) {
    write_zeros(z, blockIdx.x - blocks);
    return;
  }
  __shared__ uint32_t count[kDigits];
  if (threadIdx.x < kDigits) count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t t0 = blockIdx.x * per, t1 = min(M, t0 + per);
  for (int64_t i = t0 + threadIdx.x; i < t1; i += kSortThreads) {
    const uint32_t k = in_key != nullptr ? in_key[i] : sort_key(ids[i], V, padding);
    atomicAdd(&count[(k >> shift) & (kDigits - 1)], 1u);
  }
  __syncthreads();
  if (threadIdx.x < kDigits) hist[threadIdx.x * kMaxBlocks + blockIdx.x] = count[threadIdx.x];
}

// ... and moves its tokens to the places that follow from all of them.
__global__ __launch_bounds__(kSortThreads) void embedding_scatter_kernel(
    const int64_t* __restrict__ ids, const uint32_t* __restrict__ in_key,
    const uint32_t* __restrict__ in_tok, int64_t M, int64_t V, int64_t padding, int shift,
    int blocks, int64_t per, const uint32_t* __restrict__ hist, uint32_t* __restrict__ out_key,
    uint32_t* __restrict__ out_tok, uint32_t* __restrict__ place, Zeros z) {
  if (static_cast<int>(blockIdx.x) >= blocks) {
    write_zeros(z, blockIdx.x - blocks);
    return;
  }
  __shared__ SortLds s;
  clear_counts(s);
  uint32_t total = 0, before = 0;
  if (threadIdx.x < kDigits) {
    // (four workgroups' counts a load, all loads in flight; those past the last workgroup are not used)
    const u32x4* const row = reinterpret_cast<const u32x4*>(hist + threadIdx.x * kMaxBlocks);
    u32x4 n[kMaxBlocks / 4];
#pragma unroll
    for (int q = 0; q < kMaxBlocks / 4; ++q) n[q] = 4 * q < blocks ? row[q] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int q = 0; q < kMaxBlocks / 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int b = 4 * q + e;
        before += b < static_cast<int>(blockIdx.x) ? n[q][e] : 0u;
        total += b < blocks ? n[q][e] : 0u;
      }
    s.base[threadIdx.x] = before;
  }
  __syncthreads();
  scan_digits(s, total);
  const int64_t t0 = blockIdx.x * per, t1 = min(M, t0 + per);
  scatter_tokens(
      s, t0, t1, shift,
      [&](int64_t i, uint32_t& k, uint32_t& t) {
        if (in_key == nullptr) {
          k = sort_key(ids[i], V, padding);
          t = static_cast<uint32_t>(i);
        } else {
          k = in_key[i];
          t = in_tok[i];
        }
      },
      [&](uint32_t to, uint32_t key, uint32_t tok) {
        out_key[to] = key;
        out_tok[to] = tok;
        if (place != nullptr && key < static_cast<uint32_t>(V)) place[key] = to;
      });
}

// ---- sums ---------------------------------------------------------------------------------------

// The columns [col, col + 8) of a gradient row, read in fp32 (n of them).
template <typename G>
__device__ __forceinline__ void load_grad(const char* src, int n, float* v) {
  if (n == 8) {
    Elem<G>::unpack8(Elem<G>::template load8<true>(src), v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? Elem<G>::load1(src + j * Elem<G>::kBytes) : 0.f;
  }
}

template <typename E>
__device__ __forceinline__ void store_row(char* dst, int n, const float* v, float scale) {
  float o[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = v[j] * scale;
  if (n == 8) {
    Elem<E>::template store8<true>(dst, o);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) Elem<E>::store1(dst + j * Elem<E>::kBytes, o[j]);
  }
}

// The first `sums` workgroups: (run, column block), the run's sorted positions; the others: zeros.
// partial holds two rows of H8 floats per run: of the id that entered the run, and of the id that
// leaves it (an id that does both leaves its sum in the first).
struct Cut {
  int run;                    // positions per run
  int64_t sums;               // workgroups that add
  int col_blocks;             // per run
  int64_t zero_row0;          // rows before it were cleared with the sort
  uint32_t zero_items;        // 16-byte items (of a row) of this launch
  FastDiv per_row;            // items of a row
};

template <typename E>
__device__ __forceinline__ void zero_rows(char* dtable, const uint32_t* key, const uint32_t* place,
                                          int64_t M, int64_t H, const Cut& cut) {
  constexpr int N = 16 / Elem<E>::kBytes;
  const uint32_t i =
      static_cast<uint32_t>(blockIdx.x - cut.sums) * kEmbThreads + threadIdx.x;
  if (i >= cut.zero_items) return;
  const uint32_t r = cut.per_row.div(i);
  const int64_t row = cut.zero_row0 + r;
  const int64_t col = static_cast<int64_t>(i - r * cut.per_row.d) * N;
  if (M > 0) {
    const uint32_t p = place[row];
    if (p < M && key[p] == static_cast<uint32_t>(row)) return;
  }
  char* const to = dtable + (row * H + col) * Elem<E>::kBytes;
  if (col + N <= H) {
    st16<true>(to, u32x4{0u, 0u, 0u, 0u});
  } else {
    for (int j = 0; j < H - col; ++j) Elem<E>::store1(to + j * Elem<E>::kBytes, 0.f);
  }
}

constexpr int kSumAhead = 4;   // gradient rows in flight per thread

template <typename G, typename E>
__global__ __launch_bounds__(kEmbThreads) void embedding_write_kernel(
    const char* __restrict__ dout, const uint32_t* __restrict__ key,
    const uint32_t* __restrict__ tok, const uint32_t* __restrict__ place,
    char* __restrict__ dtable, float* __restrict__ partial, float scale, int64_t M, int64_t V,
    int64_t H, int64_t H8, Cut cut) {
  if (static_cast<int64_t>(blockIdx.x) >= cut.sums) {
    zero_rows<E>(dtable, key, place, M, H, cut);
    return;
  }
  const int64_t run = blockIdx.x / static_cast<uint32_t>(cut.col_blocks);
  const int64_t col =
      (static_cast<int64_t>(blockIdx.x % static_cast<uint32_t>(cut.col_blocks)) * kEmbThreads +
       threadIdx.x) * 8;
  if (col >= H) return;
  const int n = static_cast<int>(min(int64_t{8}, H - col));
  const int64_t p0 = run * cut.run, p1 = min(M, p0 + cut.run);
  const uint32_t none = static_cast<uint32_t>(V);
  uint32_t id = key[p0];
  if (id == none) return;                        // (and all that follow)
  bool entered = p0 > 0 && key[p0 - 1] == id;    // the sum so far continues an earlier run's
  float acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  float* const mine = partial + run * 2 * H8 + col;
  auto put_partial = [&](float* to) {
    *reinterpret_cast<f32x4*>(to) = f32x4{acc[0], acc[1], acc[2], acc[3]};
    *reinterpret_cast<f32x4*>(to + 4) = f32x4{acc[4], acc[5], acc[6], acc[7]};
  };
  auto put_row = [&]() {
    store_row<E>(dtable + (static_cast<int64_t>(id) * H + col) * Elem<E>::kBytes, n, acc, scale);
  };
  for (int64_t p = p0; p < p1; p += kSumAhead) {
    float v[kSumAhead][8];
#pragma unroll
    for (int u = 0; u < kSumAhead; ++u) {
      // (past the run: its last row, unused)
      const int64_t t = tok[min(p + u, p1 - 1)];
      load_grad<G>(dout + (t * H + col) * Elem<G>::kBytes, n, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kSumAhead; ++u) {
      if (p + u >= p1) break;
      const uint32_t k = key[p + u];
      if (k != id) {
        if (entered) put_partial(mine);
        else put_row();
        id = k;
        entered = false;
        if (k == none) return;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = acc[j] + v[u][j];
    }
  }
  const bool leaves = p1 < M && key[p1] == id;
  if (entered) put_partial(mine);
  else if (leaves) put_partial(mine + H8);
  else put_row();
}

// Workgroup (run, column block of 64 x 8): the id that leaves the run, if it began in it.  Its partial
// rows are added in run order by four groups, each a quarter of them, joined in their order.
constexpr int kJoinCols = kWave * 8;
constexpr int kJoinGroups = kEmbThreads / kWave;
template <typename E>
__global__ __launch_bounds__(kEmbThreads) void embedding_join_kernel(
    const uint32_t* __restrict__ key, const float* __restrict__ partial, char* __restrict__ dtable,
    float scale, int64_t M, int64_t V, int64_t H, int64_t H8, int run_len, int col_blocks) {
  __shared__ float sum[kJoinGroups][kJoinCols];
  const int64_t run = blockIdx.x / static_cast<uint32_t>(col_blocks);
  const int64_t p0 = run * run_len, p1 = p0 + run_len;
  if (p1 >= M) return;
  const uint32_t id = key[p1 - 1];
  if (id == static_cast<uint32_t>(V) || key[p1] != id) return;
  if (p0 > 0 && key[p0 - 1] == id) return;       // (began before: the keys are sorted)
  // one past the last position of the id
  int64_t lo = p1, hi = M;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (key[mid] <= id) lo = mid + 1;
    else hi = mid;
  }
  const int64_t last = (lo - 1) / run_len;
  const int lane = threadIdx.x % kWave, group = threadIdx.x / kWave;
  const int64_t col =
      static_cast<int64_t>(blockIdx.x % static_cast<uint32_t>(col_blocks)) * kJoinCols + lane * 8;
  const bool on = col < H;
  const int64_t per = (last - run + kJoinGroups - 1) / kJoinGroups;
  const int64_t r0 = run + 1 + group * per, r1 = min(last + 1, r0 + per);
  float acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  if (on) {
#pragma unroll 4
    for (int64_t r = r0; r < r1; ++r) {
      const f32x4* row = reinterpret_cast<const f32x4*>(partial + r * 2 * H8 + col);
      const f32x4 a = row[0], b = row[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[j] = acc[j] + a[j];
        acc[4 + j] = acc[4 + j] + b[j];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[group][lane * 8 + j] = acc[j];
  __syncthreads();
  if (group != 0 || !on) return;
  const float* first = partial + run * 2 * H8 + H8 + col;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    acc[j] = first[j];
#pragma unroll
    for (int g = 0; g < kJoinGroups; ++g) acc[j] = acc[j] + sum[g][lane * 8 + j];
  }
  store_row<E>(dtable + (static_cast<int64_t>(id) * H + col) * Elem<E>::kBytes,
               static_cast<int>(min(int64_t{8}, H - col)), acc, scale);
}

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Workspace of a backward: sorted keys and tokens twice, the histograms, the places, the partial rows.
struct Layout {
  int64_t hist, place, partial, bytes;   // byte offsets; the total
};
Layout emb_layout(int64_t M, int64_t V, int64_t H) {
  Layout l;
  l.hist = 4 * round_up(M * 4, 256);
  l.place = l.hist + int64_t{kDigits} * kMaxBlocks * 4;
  l.partial = l.place + round_up(V * 4, 256);
  const int run = run_length(M);
  l.bytes = l.partial + (M + run - 1) / run * 2 * round_up(H, 8) * 4;
  return l;
}

bool bad_sizes(int64_t M, int64_t V, int64_t H) {
  return M < 0 || V < 0 || H < 0 || V >= (int64_t{1} << 31) - 1 || M >= (int64_t{1} << 31) - 1 ||
         H > (int64_t{1} << 24);
}

}  // namespace
}  // namespace soupk

using namespace soupk;

extern "C" __attribute__((visibility("default"))) int soupk_embedding_fwd(
    const void* table, int32_t dtype, const int64_t* ids, void* out, int32_t out_dtype, float scale,
    int64_t M, int64_t V, int64_t H, void* stream) {
  if (bad_sizes(M, V, H)) return kInvalid;
  if (dtype != out_dtype && out_dtype != SOUPK_DTYPE_F32) return kInvalid;
  if (M == 0 || H == 0) return kOk;
  if (bad_elem_ptr(out, out_dtype) || !ids || (reinterpret_cast<uintptr_t>(ids) & 7u))
    return kInvalid;
  if (V > 0 && bad_elem_ptr(table, dtype)) return kInvalid;
  return with_type(dtype, [&](auto in) {
    return with_type(out_dtype, [&](auto o) -> int {
      using In = typename decltype(in)::type;
      using Out = typename decltype(o)::type;
      if constexpr (std::is_same_v<In, Out> || std::is_same_v<Out, float>) {
        const int64_t per_row = (H + lookup_cols<Out>() - 1) / lookup_cols<Out>();
        const int64_t rows_per = ((int64_t{1} << 31) - 1 - kEmbThreads) / per_row;
        const FastDiv div(static_cast<uint32_t>(per_row));
        for (int64_t r0 = 0; r0 < M; r0 += rows_per) {
          const uint32_t items = static_cast<uint32_t>(std::min(rows_per, M - r0) * per_row);
          const int rc = launch_kernel(
              embedding_fwd_kernel<In, Out>, dim3((items + kEmbThreads - 1) / kEmbThreads),
              dim3(kEmbThreads), static_cast<hipStream_t>(stream),
              // (of an empty table no row is taken; the load whose value is not used has to go
              // somewhere)
              V > 0 ? static_cast<const char*>(table) : reinterpret_cast<const char*>(out), ids,
              static_cast<char*>(out), scale, V, H, items, r0, div);
          if (rc != kOk) return rc;
        }
        return kOk;
      } else {
        return kInvalid;
      }
    });
  });
}

extern "C" __attribute__((visibility("default"))) int soupk_embedding_bwd_workspace(
    int64_t M, int64_t V, int64_t H, int64_t* bytes) {
  if (bad_sizes(M, V, H) || bytes == nullptr) return kInvalid;
  *bytes = emb_layout(M, V, H).bytes;
  return kOk;
}

extern "C" __attribute__((visibility("default"))) int soupk_embedding_bwd(
    const void* dout, int32_t grad_dtype, const int64_t* ids, void* dtable, int32_t dtype,
    float scale, int64_t padding_idx, void* workspace, int64_t workspace_bytes, int64_t M,
    int64_t V, int64_t H, void* stream) {
  if (bad_sizes(M, V, H)) return kInvalid;
  if (dtype != grad_dtype && grad_dtype != SOUPK_DTYPE_F32) return kInvalid;
  if (V == 0 || H == 0) return kOk;
  if (bad_elem_ptr(dtable, dtype)) return kInvalid;
  const Layout l = emb_layout(M, V, H);
  if (M > 0) {
    if (bad_elem_ptr(dout, grad_dtype) || !ids || (reinterpret_cast<uintptr_t>(ids) & 7u))
      return kInvalid;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) || workspace_bytes < l.bytes)
      return kInvalid;
  }
  const int64_t H8 = round_up(H, 8);
  const int run = run_length(M);
  const int64_t runs = (M + run - 1) / run;
  const int col_blocks = static_cast<int>((H8 / 8 + kEmbThreads - 1) / kEmbThreads);
  const int join_blocks = static_cast<int>((H + kJoinCols - 1) / kJoinCols);
  if (runs * join_blocks > kMaxGrid) return kInvalid;               // (>= runs * col_blocks)
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t row_bytes = H * (dtype == SOUPK_DTYPE_F32 ? 4 : 2);
  int bits = 0;
  while ((V >> bits) != 0) ++bits;
  const int passes = (bits + kDigitBits - 1) / kDigitBits;
  const bool small = M <= kOneBlock;
  const int launches = M == 0 ? 0 : small ? 1 : 2 * passes;
  // The rows cleared with the sort: a multiple of 8 per launch (whole 16-byte words).
  const int64_t hidden_rows =
      launches ? std::min<int64_t>(hidden_bytes(small) / row_bytes, V / launches) / 8 * 8 : 0;
  auto zeros = [&](int k) {
    return Zeros{static_cast<char*>(dtable) + k * hidden_rows * row_bytes,
                 hidden_rows * row_bytes / 16};
  };
  const int zero_blocks =
      static_cast<int>((hidden_rows * row_bytes / 16 + kSortThreads - 1) / kSortThreads);
  char* const ws = static_cast<char*>(workspace);
  const int64_t m4 = round_up(M * 4, 256);
  uint32_t* const key[2] = {reinterpret_cast<uint32_t*>(ws), reinterpret_cast<uint32_t*>(ws + m4)};
  uint32_t* const tok[2] = {reinterpret_cast<uint32_t*>(ws + 2 * m4),
                            reinterpret_cast<uint32_t*>(ws + 3 * m4)};
  uint32_t* const place = reinterpret_cast<uint32_t*>(ws + l.place);
  if (M > 0 && small) {
    const int rc = launch_kernel(embedding_sort_small_kernel, dim3(1 + zero_blocks),
                                 dim3(kSortThreads), s, ids, M, V, padding_idx, passes, key[0],
                                 tok[0], key[1], tok[1], place, zeros(0));
    if (rc != kOk) return rc;
  } else if (M > 0) {
    const int64_t per = round_up((M + kMaxBlocks - 1) / kMaxBlocks, kSortThreads);
    const int blocks = static_cast<int>((M + per - 1) / per);
    uint32_t* const hist = reinterpret_cast<uint32_t*>(ws + l.hist);
    for (int p = 0; p < passes; ++p) {
      const uint32_t* const in_key = p ? key[p & 1] : nullptr;
      const uint32_t* const in_tok = p ? tok[p & 1] : nullptr;
      int rc = launch_kernel(embedding_hist_kernel, dim3(blocks + zero_blocks), dim3(kSortThreads),
                             s, ids, in_key, M, V, padding_idx, p * kDigitBits, blocks, per, hist,
                             zeros(2 * p));
      if (rc != kOk) return rc;
      rc = launch_kernel(embedding_scatter_kernel, dim3(blocks + zero_blocks), dim3(kSortThreads),
                         s, ids, in_key, in_tok, M, V, padding_idx, p * kDigitBits, blocks, per,
                         static_cast<const uint32_t*>(hist), key[(p + 1) & 1], tok[(p + 1) & 1],
                         p == passes - 1 ? place : nullptr, zeros(2 * p + 1));
      if (rc != kOk) return rc;
    }
  }
  const uint32_t* const skey = key[passes & 1];
  const uint32_t* const stok = tok[passes & 1];
  float* const partial = reinterpret_cast<float*>(ws + l.partial);
  const int64_t row_items = (row_bytes + 15) / 16;
  const int64_t rows_per =
      std::max<int64_t>(1, ((int64_t{1} << 30) - kEmbThreads) / row_items);
  return with_type(grad_dtype, [&](auto gt) {
    return with_type(dtype, [&](auto et) -> int {
      using G = typename decltype(gt)::type;
      using E = typename decltype(et)::type;
      if constexpr (std::is_same_v<G, E> || std::is_same_v<G, float>) {
        // (one launch, unless the table's items do not fit 32 bits)
        int64_t row = launches * hidden_rows;
        Cut cut{run, runs * col_blocks, col_blocks, 0, 0, FastDiv(static_cast<uint32_t>(row_items))};
        do {
          const int64_t n = std::min(rows_per, V - row);
          cut.zero_row0 = row;
          cut.zero_items = static_cast<uint32_t>(n * row_items);
          const int64_t grid = cut.sums + (cut.zero_items + kEmbThreads - 1) / kEmbThreads;
          if (grid > 0) {
            const int st = launch_kernel(
                embedding_write_kernel<G, E>, dim3(static_cast<unsigned>(grid)), dim3(kEmbThreads),
                s, static_cast<const char*>(dout), skey, stok,
                static_cast<const uint32_t*>(place), static_cast<char*>(dtable), partial, scale, M,
                V, H, H8, cut);
            if (st != kOk) return st;
          }
          row += n;
          cut.sums = 0;
        } while (row < V);
        if (M == 0) return kOk;
        return launch_kernel(embedding_join_kernel<E>,
                             dim3(static_cast<unsigned>(runs * join_blocks)), dim3(kEmbThreads), s,
                             skey, static_cast<const float*>(partial), static_cast<char*>(dtable),
                             scale, M, V, H, H8, run, join_blocks);
      } else {
        return kInvalid;
      }
    });
  });
}
