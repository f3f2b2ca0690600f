// Attention of new tokens over a paged key-value cache: split over the cache's length and joined.
//
// For token i of the n_b new ones of sequence b, whose keys and values (its own included) are the first
// `length_b` positions of the cache, and query head h with key head h / G:
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m),  j <= length_b - n_b + i
// m is a running reference value (raised when a score exceeds it by more than a margin, 8 in bf16 as in the training
// attention: weights of 2^8), sums and products in fp32; a token that sees no key gets zeros.
//
// What bounds it: the cache's bytes -- a key head's row is read once for the G query heads and the few new
// tokens that share it.  So the query rows of a key head (row = token * G + head in the group, 16 * NB of
// them a tile) are the 16 columns of v_mfma_f32_16x16x32 products, and keys its rows:
//   S^T (32 keys x 16 rows) = K Q^T        A = K rows staged in LDS
//   O^T (D x 16 rows) += V^T P^T           A = V^T by transpose reads of rows staged in LDS
// An operand is of the cache's type, so P goes in as two: rounded, and what that left, rounded again (a relative
// error of 2^-16 in bf16, 2^-22 in fp16).  Rounded alone it added as much error again, in squares, as the output's own
// rounding.  MI355X, with the second product / without: 64 sequences of up to 8192 keys 172.0 / 171.5 us, one
// token over 32768 keys 14.1 / 14.0, 5 new tokens of 16 sequences 20.8 / 19.9, of 32 of up to 8192 keys 64.4 / 60.8, 64
// tokens of 8 sequences 93 / 82.
// A wavefront is on its own inside a chunk: it owns 32 of the chunk's 128 keys, its own strip of LDS and its
// own softmax state; the four are merged once, at the end of an item or part.  No barrier is in the
// loop.  Page numbers are read two chunks ahead and rows one chunk ahead of their use.
//
// Split: the work is the list of all chunks of all items -- (sequence, key head, row tile) -- in that order,
// cut into equal parts, one a workgroup: a long sequence among short ones, or one alone, fills the chip the same
// way, whatever the lengths are (they are in device memory: a captured graph's replays may change
// them; cut_of() says where it does not).  Where the items are few, each is cut for itself (a workgroup that crosses into another item waits
// for queries, page numbers and rows once more); where they are many, a part may end one item and
// begin others.  A workgroup writes what lies whole inside its part; of an item that reaches across an end it
// leaves the unnormalised sum, its reference value and its weight, two at most, and a second launch
// joins those in workgroup order: the same bits every time.
//
// MI355X: 64 sequences of up to 8192 keys, 8 heads of 128 in bf16 (1.09 GB) 169 us and a join of 4.7: 6.5 TB/s.  A
// single step is latency: lengths and schedule 1.2 us, page numbers and queries 1, rows 2.4, a wavefront's 32 keys
// 1, merge 1; the join 4 (8 sequences of up to 4096 keys 12.3 us in all).

#include <algorithm>
#include <type_traits>

#include "elem.hpp"
#include "fastdiv.hpp"

namespace soupk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kWaveKeys = 32;
constexpr int kChunk = kWaves * kWaveKeys;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

// kRaise: how far below the largest score the reference value is set, kMost: by how much a score may exceed it (log2 of
// a weight).  fp16 weights go up to 2^15, so that those without all bits begin at 2^-27 of the largest (with 0 and 8:
// at 2^-14, and 8000 weights of 2^-25 beside one of 1 were lost).
template <typename T>
struct Ops;
template <>
struct Ops<f16> {
  static constexpr float kRaise = 13.f, kMost = 15.f;
  static constexpr uint16_t kNoNumber = 0x7c00;     // (bits of infinities and NaN)
  typedef f16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f4 mfma(u32x4 a, u32x4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0,
                                                  0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_h2(a, b); }
  static __device__ __forceinline__ float first(uint32_t w) { return lo_h(w); }
  static __device__ __forceinline__ float second(uint32_t w) { return hi_h(w); }
};
template <>
struct Ops<bf16> {
  static constexpr float kRaise = 0.f, kMost = 8.f;
  static constexpr uint16_t kNoNumber = 0x7f80;
  typedef bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f4 mfma(u32x4 a, u32x4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0,
                                                   0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_b2(a, b); }
  static __device__ __forceinline__ float first(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float second(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};

struct PagedArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* cu;          // null: one new token a sequence
  uint16_t* out;
  uint32_t* first;            // [B + 3]: first chunk of each sequence, their number, a part's, an item's multiple
  float* part;                // two of a workgroup: rows x D sums, rows reference values, rows weights
  int64_t rows, q_stride, max_pages, pages, page_stride;
  int B, NKV, G, D, page_size, parts;
  int held;                   // keys that a row of the block table holds (at most 2^30)
  bool tiled;                 // more than one row tile a sequence
  float scale_log2;
  FastDiv by_page, by_group, by_quad;
};

// Sequence b's rows and length, which may pass its block table: its tokens' places count from it all the same.
// One whose bounds leave the rows has no keys, so that the rows which it spans get their zeros as any row
// without keys does.
struct Seq {
  int start, news, len;
};
__device__ __forceinline__ Seq sequence(const PagedArgs& p, int b) {
  int s0 = b, s1 = b + 1;
  if (p.cu != nullptr) {
    s0 = p.cu[b];
    s1 = p.cu[b + 1];
  }
  const int rows = static_cast<int>(p.rows);      // (at most 2^23)
  const bool ok = s0 >= 0 && s1 <= rows;
  s0 = min(max(s0, 0), rows);
  s1 = min(max(s1, s0), rows);
  return {s0, s1 - s0, ok ? max(p.lengths[b], 0) : 0};
}
// Chunks of a (key head, row tile) of a sequence (one at least, which writes the zeros of one without
// keys), and its row tiles.
__device__ __forceinline__ int chunks_of(const Seq& s, int held) {
  return max((min(s.len, held) + kChunk - 1) / kChunk, 1);
}
template <int R>
__device__ __forceinline__ int tiles_of(const Seq& s, int G) { return (s.news * G + R - 1) / R; }

// Max (of a NaN: NaN) / sum over the four lanes that share a row (lane % 16).
__device__ __forceinline__ float column_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __builtin_elementwise_maximum(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Inclusive sum over the wavefront's lanes, and over the workgroup's threads, in order.
// (Of lanes by DPP: within rows of 16 from 1, 2, 4 and 8 lanes before, then the last lane of a row for the next
// one and of the first half for the second.)
__device__ __forceinline__ uint32_t scan_lanes(uint32_t v) {
  auto add = [&](auto ctrl, auto rows) {
    v += __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
  };
  using std::integral_constant;
  constexpr integral_constant<int, 0xf> all;
  add(integral_constant<int, 0x111>{}, all);
  add(integral_constant<int, 0x112>{}, all);
  add(integral_constant<int, 0x114>{}, all);
  add(integral_constant<int, 0x118>{}, all);
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return v;
}
__device__ __forceinline__ uint32_t scan_threads(uint32_t v, uint32_t* sums, uint32_t& total) {
  const int w = threadIdx.x >> 6;
  v = scan_lanes(v);
  if ((threadIdx.x & 63) == 63) sums[w] = v;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) before += sums[i];
    total += sums[i];
  }
  __syncthreads();
  return before + v;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int l) { return __builtin_amdgcn_readlane(v, l); }

// A barrier of the workgroup for what is in LDS (global stores stay in flight).
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// How the list is cut: chunks of a part, and what an item's chunks are rounded up to.
// (Cut for themselves, items are given a part more each, whether they fill it or not: close to half as many items as
// parts, a part is up to twice the mean.  16 sequences of up to 16 tokens and 8192 keys, 32/8 heads: 240 items of 8032
// chunks in all, 30 a part of 512, 15.7 their mean; 119 us, for 43 of memory.)
struct Cut {
  uint32_t per, unit;
};
__device__ __forceinline__ Cut cut_of(uint32_t chunks, uint32_t items, uint32_t parts) {
  if (2 * items <= parts) {       // each item for itself: sum of ceil(chunks / per) <= chunks / per + items
    const uint32_t per = max((chunks + (parts - items) - 1) / (parts - items), 1u);
    return {per, per};
  }
  return {max((chunks + parts - 1) / parts, 1u), 1};
}
__device__ __forceinline__ uint32_t rounded(uint32_t n, uint32_t unit) {
  return unit == 1 ? n : (n + unit - 1) / unit * unit;
}

// A wavefront's 32 keys of a chunk, as loaded: 16-byte pieces of whole rows (a cache line at once: in the
// operands' own order an instruction would touch half a line of 16 rows), and which keys have a place.
template <int N>
struct Rows {
  u32x4 k[N], v[N];
  uint32_t ok;
};

template <typename T, int DP, int NB>
struct Tile {
  static constexpr int S = DP / 32, DT = DP / 16, R = 16 * NB;
  // Queries in LDS for 32 rows of a wide head, whose accumulators leave them no registers (in registers, 5 new
  // tokens of 32 sequences of up to 8192 keys took 73.2 us instead of 68.7, of 8 sequences of up to 4096 20.1 / 17.3).
  static constexpr bool kQueriesInLds = NB == 2 && DP == 128;
  // Rows in LDS: reads of 16 and 8 bytes free of conflicts with 16 halves between them, and two workgroups a CU
  // beside the queries with 8.
  static constexpr int kLd = kQueriesInLds ? DP + 8 : DP + 16;
  static constexpr int kStrip = 2 * kWaveKeys * kLd;         // halves of a wavefront's strip: K, then V
  // a load instruction takes kPer whole rows, kLanes lanes each (of them D / 8 with pieces of their own)
  static constexpr int kLanes = DP / 8, kPer = kWave / kLanes, kLoads = (kWaveKeys + kPer - 1) / kPer;
};

// PAST: keys and values are read past the caches.
template <typename T, int DP, int NB, bool PAST>
__global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) void paged_attention_kernel(PagedArgs p) {
  using TL = Tile<T, DP, NB>;
  constexpr int S = TL::S, DT = TL::DT, R = TL::R, kLd = TL::kLd;
  constexpr int kSumLd = DP + 4;          // floats of a row of the merge
  // (the merge of the wavefronts takes the strips over)
  static_assert(TL::kStrip * 2 >= R * kSumLd * 4, "");
  __shared__ __align__(16) uint16_t strips[kWaves * TL::kStrip];
  __shared__ float stats[kWaves][2][16 * NB];
  __shared__ __align__(16) uint16_t q_rows[TL::kQueriesInLds ? R * kLd : 8];
  __shared__ uint32_t sums[kWaves];
  __shared__ uint32_t found[2];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, ql = lane & 15, gr = lane >> 4;
  const int D = p.D;

  // ---- this workgroup's part of the list, and the sequence that it begins in
  Cut cut;
  uint32_t c_begin, c_end, seq0 = 0;
  int b = p.B;
  // (Workgroups go round the eight XCDs.  Row tiles of a sequence, which stand next to each other in the list and
  // read the same keys, go to one of them: 8 sequences' 64 new tokens of 32 heads over 4096 keys 99 us instead of
  // 165.  Items that are cut for themselves are many parts apart: there it cost more than it gave.)
  uint32_t me = blockIdx.x;
  auto part_of = [&](uint32_t total) {
    const uint32_t used = p.tiled && cut.unit == 1 ? (total + cut.per - 1) / cut.per : 0;
    const uint32_t xcd = blockIdx.x & 7;
    me = blockIdx.x < used ? xcd * (used >> 3) + min(xcd, used & 7) + (blockIdx.x >> 3) : blockIdx.x;
    c_begin = min(me * cut.per, total);
    c_end = min(c_begin + cut.per, total);
  };
  Seq lane_seq{0, 0, 0};          // (up to 64 sequences: each lane has one)
  if (p.B <= kWave) {             // every wavefront for itself
    uint32_t items = 0, chunks = 0;
    if (lane < p.B) {
      const Seq s = sequence(p, lane);
      lane_seq = s;
      items = static_cast<uint32_t>(tiles_of<R>(s, p.G)) * p.NKV;
      chunks = chunks_of(s, p.held);
    }
    cut = cut_of(lane_of(scan_lanes(items * chunks), 63), lane_of(scan_lanes(items), 63), p.parts);
    const uint32_t n = items * rounded(chunks, cut.unit), upto = scan_lanes(n), total = lane_of(upto, 63);
    part_of(total);
    const uint64_t at = __ballot(c_begin >= upto - n && c_begin < upto);
    if (at != 0) {
      b = __ffsll(static_cast<unsigned long long>(at)) - 1;
      seq0 = lane_of(upto - n, b);
    }
    if (blockIdx.x == 0 && w == 0) {
      if (lane < p.B) p.first[lane] = upto - n;
      if (lane == 0) {
        p.first[p.B] = total;
        p.first[p.B + 1] = cut.per;
        p.first[p.B + 2] = cut.unit;
      }
    }
  } else {
    uint32_t total = 0, all_chunks = 0, all_items = 0;
    if (threadIdx.x == 0) found[0] = p.B;
    auto look = [&](int q, uint32_t& items, uint32_t& chunks) {
      items = chunks = 0;
      if (q >= p.B) return;
      const Seq s = sequence(p, q);
      items = static_cast<uint32_t>(tiles_of<R>(s, p.G)) * p.NKV;
      chunks = chunks_of(s, p.held);
    };
    uint32_t items, chunks;
    for (int q = threadIdx.x; q < p.B; q += kThreads) {
      look(q, items, chunks);
      all_chunks += items * chunks;
      all_items += items;
    }
    scan_threads(all_chunks, sums, all_chunks);
    scan_threads(all_items, sums, all_items);
    cut = cut_of(all_chunks, all_items, p.parts);
    for (int pass = 0;; ++pass) {
      uint32_t before = 0;
      for (int b0 = 0; b0 < p.B; b0 += kThreads) {
        const int q = b0 + static_cast<int>(threadIdx.x);
        look(q, items, chunks);
        uint32_t sum;
        const uint32_t n = items * rounded(chunks, cut.unit), upto = before + scan_threads(n, sums, sum);
        before += sum;
        if (pass == 0 && blockIdx.x == 0 && q < p.B) p.first[q] = upto - n;
        if (p.B <= kThreads) total = sum;
        part_of(total);
        if (c_begin >= upto - n && c_begin < upto) {
          found[0] = q;
          found[1] = upto - n;
        }
      }
      total = before;
      if (p.B <= kThreads || pass == 1) break;      // (more sequences than threads: once the total is known)
    }
    part_of(total);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      p.first[p.B] = total;
      p.first[p.B + 1] = cut.per;
      p.first[p.B + 2] = cut.unit;
    }
    __syncthreads();
    b = static_cast<int>(found[0]);
    seq0 = found[1];
  }
  // rows that belong to no sequence
  if (p.cu != nullptr) {
    const int64_t lead = min(max(static_cast<int64_t>(p.cu[0]), int64_t{0}), p.rows);
    const int64_t tail = min(max(static_cast<int64_t>(p.cu[p.B]), lead), p.rows);
    const int64_t width = static_cast<int64_t>(p.NKV) * p.G * D;
    for (int64_t r = blockIdx.x; r < lead + p.rows - tail; r += gridDim.x) {
      uint16_t* o = p.out + (r < lead ? r : tail + r - lead) * width;
      for (int64_t c = threadIdx.x; c < width; c += kThreads) o[c] = 0;
    }
  }
  uint16_t* const strip = strips + w * TL::kStrip;
  // this lane's piece of a row, and its row of load i (lanes and rows too many repeat the last ones)
  const int lane_row = min(lane / TL::kLanes, TL::kPer - 1);
  auto piece_of = [&](int l) { return 8 * min(l - l / TL::kLanes * TL::kLanes, D / 8 - 1); };
  const int piece = piece_of(lane);
  auto row_of = [&](int i) {
    const int row = i * TL::kPer + lane_row;
    return kWaveKeys % TL::kPer ? min(row, kWaveKeys - 1) : row;
  };
  // of the sums of the merge: this thread's columns, first row and rows at a time
  const int sum_row = p.by_quad.div(threadIdx.x), sum_col = 4 * (threadIdx.x - sum_row * p.by_quad.d);
  const int sum_rows = p.by_quad.div(kThreads);
  uint32_t c = c_begin;
  while (c < c_end && b < p.B) {
    const Seq sq = p.B > kWave ? sequence(p, b)
                               : Seq{__builtin_amdgcn_readlane(lane_seq.start, b),
                                     __builtin_amdgcn_readlane(lane_seq.news, b),
                                     __builtin_amdgcn_readlane(lane_seq.len, b)};
    const uint32_t chunks = chunks_of(sq, p.held), tiles = tiles_of<R>(sq, p.G), span = rounded(chunks, cut.unit);
    const uint32_t seq_chunks = span * tiles * p.NKV;
    if (c >= seq0 + seq_chunks) {         // (the sequence is done, or has no rows)
      seq0 += seq_chunks;
      ++b;
      continue;
    }
    const uint32_t item = (c - seq0) / span;
    const int h = tiles == 1 ? item : item / tiles, tile = item - h * tiles;
    const uint32_t item0 = seq0 + item * span;
    const int j_begin = c - item0;
    const int j_end = min(chunks, c_end - item0);
    c = item0 + span;                     // (what is left of it, if anything, is the next workgroup's)

    // (the first row of the tile sees the fewest keys, the last one the most)
    const int rr0 = tile * R, rr1 = min(rr0 + R, sq.news * p.G) - 1;
    auto seen_by = [&](int rr) {
      return min(max(sq.len - sq.news + static_cast<int>(p.by_group.div(rr)) + 1, 0), p.held);
    };
    const int seen_all = seen_by(rr0), seen_any = seen_by(rr1);

    const int32_t* pages = p.table + static_cast<int64_t>(b) * p.max_pages;
    // the page of key `lane % 32` of this wavefront's in chunk j (of the last key for those behind it), as it is in
    // the table: looked at when its rows are loaded, as a wait for it is one for all loads before it
    auto find = [&](int j) { return pages[p.by_page.div(min(j * kChunk + w * kWaveKeys + (lane & 31), seen_any - 1))]; };
    // (Places worked out here where registers are few: kept over all items, they would be kept in memory, and a wait
    // for one is a wait for all loads before it.)
    int here = lane;
    if constexpr (NB == 2) __asm__ volatile("" : "+v"(here));
    const int64_t lane_at = static_cast<int64_t>(h) * p.page_size * D + piece_of(here);
    const uint16_t* const k_lane = p.k + lane_at;
    const uint16_t* const v_lane = p.v + lane_at;
    auto load = [&](Rows<TL::kLoads>& r, int found_page, int j) {
      const int key = j * kChunk + w * kWaveKeys + (lane & 31);
      if (found_page >= p.pages || key >= seen_any) found_page = -1;
      r.ok = static_cast<uint32_t>(__ballot(found_page >= 0));
      // (a key without a place reads a row of page 0: masked, and its value zeroed, below)
      const int slot = key - static_cast<int>(p.by_page.div(key)) * p.page_size;
      const int64_t at = static_cast<int64_t>(max(found_page, 0)) * p.page_stride + static_cast<int64_t>(slot) * D;
      const int at_lo = static_cast<int>(at), at_hi = static_cast<int>(at >> 32);
#pragma unroll
      for (int i = 0; i < TL::kLoads; ++i) {
        const int row = row_of(i);
        const uint32_t lo = __shfl(at_lo, row), hi = __shfl(at_hi, row);
        const int64_t to = static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
        r.k[i] = ld<PAST>(reinterpret_cast<const u32x4*>(k_lane + to));
        r.v[i] = ld<PAST>(reinterpret_cast<const u32x4*>(v_lane + to));
      }
    };
    if (D < DP) {                         // columns past D: zeros of K, which meet any of Q, and of V
      for (int e = lane; e < 2 * kWaveKeys * (DP - D) / 8; e += kWave) {
        const int row = e & (2 * kWaveKeys - 1);
        *reinterpret_cast<u32x4*>(strip + row * kLd + D + 8 * (e / (2 * kWaveKeys))) = u32x4{0, 0, 0, 0};
      }
    }
    // (chunks in which this wavefront has keys that the tile sees)
    const int j_mine = min(j_end, (seen_any - w * kWaveKeys + kChunk - 1) / kChunk);
    Rows<TL::kLoads> r;
    int next;                             // (not set before: that would wait for the last item's stores)
    if (j_begin < j_mine) next = find(j_begin);
    // ---- the query rows, on their way while the page numbers are
    // (for LDS, a wavefront loads every fourth piece; pieces too many repeat the last one)
    constexpr int kParts = (NB * S + kWaves - 1) / kWaves;
    u32x4 qf[NB][S], q_part[kParts];
    auto part_at = [&](int i) { return min(w + i * kWaves, NB * S - 1); };
    int limit[NB];                        // keys that this lane's row sees
    const int q_row = here & 15, q_col = 8 * (here >> 4);
    // (rows too many repeat the last one, and columns past D the first, which meet zeros of K)
    auto query = [&](int u, int s) {
      const int rr = min(rr0 + 16 * u + q_row, rr1), i = p.by_group.div(rr), g = rr - i * p.G, d = 32 * s + q_col;
      const uint16_t* row = p.q + static_cast<int64_t>(sq.start + i) * p.q_stride + static_cast<int64_t>(h * p.G + g) * D;
      return ld16<false>(row + (d < D ? d : 0));
    };
#pragma unroll
    for (int u = 0; u < NB; ++u)
      limit[u] = seen_by(min(rr0 + 16 * u + ql, rr1));
    if constexpr (TL::kQueriesInLds) {
#pragma unroll
      for (int i = 0; i < kParts; ++i) q_part[i] = query(part_at(i) / S, part_at(i) % S);
    } else {
#pragma unroll
      for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int s = 0; s < S; ++s) qf[u][s] = query(u, s);
    }
    if (j_begin < j_mine) {
      load(r, next, j_begin);
      if (j_begin + 1 < j_mine) next = find(j_begin + 1);
    }
    if constexpr (TL::kQueriesInLds) {
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const int f = part_at(i);
        *reinterpret_cast<u32x4*>(q_rows + (16 * (f / S) + q_row) * kLd + 32 * (f % S) + q_col) = q_part[i];
      }
      lds_barrier();
    }
    f4 acc[NB][DT];
    float m_ref[NB], lsum[NB];
    auto begin = [&] {
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        m_ref[u] = -INFINITY;
        lsum[u] = 0.f;
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[u][t] = f4{0.f, 0.f, 0.f, 0.f};
      }
    };
    begin();
    // (wait for the queries here: the loop would wait for them, and for the rows that it loads, in every step)
    if constexpr (!TL::kQueriesInLds) {
#pragma unroll
      for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int s = 0; s < S; ++s) __asm__ volatile("" : "+v"(qf[u][s]));
    }
    auto chunk = [&](auto careful, int j) {
      const int key0 = j * kChunk + w * kWaveKeys;
      const uint32_t ok = r.ok;
      const bool whole = ok == ~0u;
      if (!whole) {
#pragma unroll
        for (int i = 0; i < TL::kLoads; ++i) r.v[i] = r.v[i] & (0u - ((ok >> row_of(i)) & 1));
      }
#pragma unroll
      for (int i = 0; i < TL::kLoads; ++i) {
        const int row = row_of(i);
        *reinterpret_cast<u32x4*>(strip + row * kLd + piece) = r.k[i];
        *reinterpret_cast<u32x4*>(strip + (kWaveKeys + row) * kLd + piece) = r.v[i];
      }
      // the next chunk's rows, and the page numbers of the one after it
      if (j + 1 < j_mine) {
        load(r, next, j + 1);
        if (j + 2 < j_mine) next = find(j + 2);
      }
      __asm__ volatile("" ::: "memory");
      f4 sc[NB][2];
#pragma unroll
      for (int u = 0; u < NB; ++u) sc[u][0] = sc[u][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const u32x4 kf = *reinterpret_cast<const u32x4*>(strip + (16 * n + ql) * kLd + 32 * s + 8 * gr);
#pragma unroll
          for (int u = 0; u < NB; ++u) {
            u32x4 q = qf[u][s];
            if constexpr (TL::kQueriesInLds)
              q = *reinterpret_cast<const u32x4*>(q_rows + (16 * u + ql) * kLd + 32 * s + 8 * gr);
            sc[u][n] = Ops<T>::mfma(kf, q, sc[u][n]);
          }
        }
      }
      u32x4 pb[NB], rest[NB];               // the weights rounded, and what is left of them
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        sc[u][0] = sc[u][0] * p.scale_log2;
        sc[u][1] = sc[u][1] * p.scale_log2;
        if (!whole || key0 + kWaveKeys > seen_all) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at = 4 * gr + (e & 3), n = e >> 2;
            const bool seen = key0 + 16 * n + at < limit[u] && ((ok >> (16 * n + at)) & 1);
            sc[u][n][e & 3] = seen ? sc[u][n][e & 3] : -INFINITY;
          }
        }
        float mx = sc[u][0][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = __builtin_elementwise_maximum(mx, sc[u][e >> 2][e & 3]);
        if (__any(!(mx - m_ref[u] <= Ops<T>::kMost))) {         // (a NaN raises it to NaN)
          // (from 2^22 on a score is no longer sure to hold the difference, and the reference value is the score)
          const float top = column_max(mx), less = __builtin_fabsf(top) < 0x1p22f ? Ops<T>::kRaise : 0.f;
          const float m_new = __builtin_elementwise_maximum(m_ref[u], top - less);
          const float alpha = m_ref[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_ref[u] - m_new);
          lsum[u] *= alpha;
#pragma unroll
          for (int t = 0; t < DT; ++t) acc[u][t] = acc[u][t] * alpha;
          m_ref[u] = m_new;
        }
        const float m_use = m_ref[u] == -INFINITY ? 0.f : m_ref[u];
        float pr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pr[e] = __builtin_amdgcn_exp2f(sc[u][e >> 2][e & 3] - m_use);
          lsum[u] += pr[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t two = Ops<T>::pack(pr[2 * e], pr[2 * e + 1]);
          pb[u][e] = two;
          rest[u][e] = Ops<T>::pack(pr[2 * e] - Ops<T>::first(two), pr[2 * e + 1] - Ops<T>::second(two));
        }
      }
      if constexpr (decltype(careful)::value) {      // (such values are added to the rows that see them)
#pragma unroll 1
        for (int key = 0; key < kWaveKeys; ++key) {
#pragma unroll
          for (int t = 0; t < DT; ++t) {
            uint16_t* at = strip + (kWaveKeys + key) * kLd + 16 * t + 4 * gr;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint16_t v = at[e];
              if ((v & Ops<T>::kNoNumber) != Ops<T>::kNoNumber) continue;
#pragma unroll
              for (int u = 0; u < NB; ++u)
                if (key0 + key < limit[u]) acc[u][t][e] += Ops<T>::first(v);
              at[e] = 0;
            }
          }
        }
      }
      __asm__ volatile("" ::: "memory");      // (no reads of V before their time: registers)
      // O^T += V^T P^T: transpose reads (lane k of a 16-lane group reads 8 bytes of row 4 gr + k / 4 at
      // column 4 (k % 4); lane i gets column i of the four rows), rows 4 gr .. + 3 and 16 more
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const uint16_t* at = strip + (kWaveKeys + 4 * gr + (ql >> 2)) * kLd + 16 * t + 4 * (ql & 3);
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at));
        const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 16 * kLd));
        const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
        const u32x4 vf = {l2.x, l2.y, h2.x, h2.y};
#pragma unroll
        for (int u = 0; u < NB; ++u) {
          acc[u][t] = Ops<T>::mfma(vf, pb[u], acc[u][t]);
          acc[u][t] = Ops<T>::mfma(vf, rest[u], acc[u][t]);
        }
      }
    };
    for (int j = j_begin; j < j_mine; ++j) chunk(std::false_type{}, j);
    // Sums that are no numbers are made again without the values that are none: 0 times one would reach the rows that
    // do not see its key, and what rounding left of a weight would turn an infinity into a NaN.
    float top[2] = {0.f, 0.f};            // (of a NaN: NaN)
    auto larger = [](float a, float b) { return __builtin_elementwise_maximum(a, __builtin_fabsf(b)); };
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) top[e >> 1] = larger(top[e >> 1], acc[u][t][e]);
    if (__any(!(larger(top[0], top[1]) < INFINITY))) {
      begin();
      load(r, find(j_begin), j_begin);
      if (j_begin + 1 < j_mine) next = find(j_begin + 1);
      for (int j = j_begin; j < j_mine; ++j) chunk(std::true_type{}, j);
    }

    // ---- the four wavefronts' sums into one
    const int real_rows = min(R, sq.news * p.G - tile * R);
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      lsum[u] = column_sum(lsum[u]);
      if (gr == 0) {
        stats[w][0][16 * u + ql] = m_ref[u];
        stats[w][1][16 * u + ql] = lsum[u];
      }
    }
    const bool complete = j_begin == 0 && j_end == static_cast<int>(chunks);
    float* const part = p.part + (2 * static_cast<int64_t>(me) + (j_begin == 0 ? 1 : 0)) * (R * (D + 2));
    float* const mine = reinterpret_cast<float*>(strip);
    lds_barrier();                      // (stats are written; the strips' last readers are done)
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      if (16 * u + ql >= real_rows) break;
      float m_all = stats[0][0][16 * u + ql];
#pragma unroll
      for (int i = 1; i < kWaves; ++i) m_all = fmaxf(m_all, stats[i][0][16 * u + ql]);
      const float f = m_ref[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_ref[u] - m_all);
      if (gr == 0) stats[w][1][16 * u + ql] = lsum[u] * f;
#pragma unroll
      for (int t = 0; t < DT; ++t)
        *reinterpret_cast<f4*>(mine + (16 * u + ql) * kSumLd + 16 * t + 4 * gr) = acc[u][t] * f;
    }
    lds_barrier();
    // a thread: four neighbouring columns of a row
    for (int rt = sum_row; rt < real_rows && sum_row < sum_rows; rt += sum_rows) {
      f4 x = f4{0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        x = x + *reinterpret_cast<const f4*>(reinterpret_cast<const float*>(strips + i * TL::kStrip) + rt * kSumLd +
                                             sum_col);
        l += stats[i][1][rt];
      }
      if (complete) {
        const int rr = tile * R + rt, i = p.by_group.div(rr), g = rr - i * p.G;
        const float inv = l == 0.f ? 0.f : 1.f / l;       // (no key: no weight)
        uint16_t* o = p.out + (static_cast<int64_t>(sq.start + i) * p.NKV + h) * p.G * D + g * D + sum_col;
        *reinterpret_cast<u32x2_a2*>(o) = u32x2{Ops<T>::pack(x[0] * inv, x[1] * inv), Ops<T>::pack(x[2] * inv, x[3] * inv)};
      } else {
        *reinterpret_cast<f4*>(part + rt * D + sum_col) = x;
        if (sum_col == 0) {
          float m = stats[0][0][rt];
#pragma unroll
          for (int i = 1; i < kWaves; ++i) m = fmaxf(m, stats[i][0][rt]);
          part[R * D + rt] = m;
          part[R * D + R + rt] = l;
        }
      }
    }
    if (c < c_end) lds_barrier();         // (the strips and stats are free again)
  }
}

// Joins the parts of the rows that reach across workgroups: one workgroup a (token, query head) and 32
// columns, 16 lanes a part.
constexpr int kJoinCols = 32;
template <typename T, int R, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_join_kernel(PagedArgs p) {
  constexpr int kJoinWaves = THREADS / kWave;
  __shared__ f4 sums[kJoinWaves * 16];      // of a wavefront: two columns' sums, weight, reference value
  const int heads = p.NKV * p.G;
  const int64_t row = blockIdx.x / heads;
  const int head = static_cast<int>(blockIdx.x - row * heads), h = head / p.G, g = head - h * p.G;
  int b = static_cast<int>(row);
  if (p.cu != nullptr) {
    int hi = p.B;                          // the last sequence that starts at or before the row
    b = 0;
    while (hi - b > 1) {
      const int mid = (b + hi) / 2;
      if (p.cu[mid] <= row) b = mid;
      else hi = mid;
    }
  }
  const Seq s = sequence(p, b);
  const uint32_t first = p.first[b], total = p.first[p.B], per = p.first[p.B + 1], unit = p.first[p.B + 2];
  if (row < s.start || row >= s.start + s.news || total == 0) return;
  const int rr = static_cast<int>(row - s.start) * p.G + g;
  const uint32_t chunks = chunks_of(s, p.held), tiles = tiles_of<R>(s, p.G);
  const uint32_t c0 = first + (h * tiles + rr / R) * rounded(chunks, unit), c1 = c0 + chunks - 1;
  const uint32_t w0 = c0 / per, w1 = c1 / per;
  if (w0 == w1 || w1 >= static_cast<uint32_t>(p.parts)) return;      // (written whole)
  const int rt = rr % R, D = p.D, lane = threadIdx.x & 63, w = threadIdx.x >> 6, ql = lane & 15;
  const int n = static_cast<int>(w1 - w0) + 1, col = blockIdx.y * kJoinCols + 2 * ql;
  const int at = min(col, D - 2);
  // every (THREADS / 16)-th part, under a reference value of the lane's own
  float x = 0.f, y = 0.f, l = 0.f, m = -INFINITY;
#pragma unroll 4
  for (int i = threadIdx.x / 16; i < n; i += THREADS / 16) {
    const float* src = p.part + (2 * static_cast<int64_t>(w0 + i) + (i == 0 ? 1 : 0)) * (R * (D + 2));
    const float mi = src[R * D + rt], li = src[R * D + R + rt];
    const float2 v = *reinterpret_cast<const float2*>(src + rt * D + at);
    const float m_new = __builtin_elementwise_maximum(m, mi);
    const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
    const float f = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - m_new);
    x = x * a + v.x * f;
    y = y * a + v.y * f;
    l = l * a + li * f;
    m = m_new;
  }
  auto join = [&] {                        // the four lanes of a column pair into one
    const float m_new = column_max(m);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
    x = column_sum(x * f);
    y = column_sum(y * f);
    l = column_sum(l * f);
    m = m_new;
  };
  join();
  if constexpr (kJoinWaves > 1) {
    if (lane < 16) sums[w * 16 + ql] = f4{x, y, l, m};
    __syncthreads();
    if (w != 0) return;
    x = y = l = 0.f;
    m = -INFINITY;
#pragma unroll
    for (int i = lane / 16; i < kJoinWaves; i += 4) {
      const f4 o = sums[i * 16 + ql];
      const float m_new = __builtin_elementwise_maximum(m, o.w);
      const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
      const float f = o.w == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(o.w - m_new);
      x = x * a + o.x * f;
      y = y * a + o.y * f;
      l = l * a + o.z * f;
      m = m_new;
    }
    join();
  }
  if (lane >= 16 || col >= D) return;
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
  *reinterpret_cast<uint32_t*>(p.out + (row * heads + head) * D + col) = Ops<T>::pack(x * inv, y * inv);
}

// The same where items are many and few of them reach across a workgroup's end: a workgroup joins the item that
// begins in the part of the main launch's workgroup of its number, if that one did not finish it.
template <typename T, int R>
__global__ __launch_bounds__(kThreads) void paged_join_last_kernel(PagedArgs p) {
  const uint32_t total = p.first[p.B], per = p.first[p.B + 1], unit = p.first[p.B + 2];
  const uint32_t c0 = blockIdx.x * per, c1 = c0 + per;
  if (c1 >= total) return;
  // the sequence of chunk c1 - 1: the last one whose first chunk is not behind it, 64 at a time
  const int lane = threadIdx.x & 63;
  int b = 0, n_left = p.B;
  while (n_left > 1) {
    const int step = (n_left + kWave - 1) / kWave, at = b + lane * step;
    const int count = __popcll(__ballot(lane * step < n_left && at < p.B && p.first[at] <= c1 - 1));
    b += (max(count, 1) - 1) * step;
    n_left = min(step, p.B - b);
    if (step == 1) break;
  }
  const Seq s = sequence(p, b);
  const uint32_t chunks = chunks_of(s, p.held), tiles = tiles_of<R>(s, p.G), span = rounded(chunks, unit);
  const uint32_t seq0 = p.first[b], item = (c1 - 1 - seq0) / span, item0 = seq0 + item * span;
  if (item0 < c0 || item0 + chunks <= c1 || item >= tiles * p.NKV) return;
  const uint32_t w1 = (item0 + chunks - 1) / per;
  if (w1 >= static_cast<uint32_t>(p.parts)) return;
  const int h = item / tiles, tile = item - h * tiles, n = static_cast<int>(w1 - blockIdx.x) + 1, D = p.D;
  const int rows = min(R, s.news * p.G - tile * R), pairs = D / 2;
  for (int e = threadIdx.x; e < rows * pairs; e += kThreads) {
    const int rt = e / pairs, col = 2 * (e - rt * pairs);
    float x = 0.f, y = 0.f, l = 0.f, m = -INFINITY;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float* src = p.part + (2 * static_cast<int64_t>(blockIdx.x + i) + (i == 0 ? 1 : 0)) * (R * (D + 2));
      const float mi = src[R * D + rt], li = src[R * D + R + rt];
      const float2 v = *reinterpret_cast<const float2*>(src + rt * D + col);
      const float m_new = __builtin_elementwise_maximum(m, mi);
      const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
      const float f = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - m_new);
      x = x * a + v.x * f;
      y = y * a + v.y * f;
      l = l * a + li * f;
      m = m_new;
    }
    const int rr = tile * R + rt, i = p.by_group.div(rr), g = rr - i * p.G;
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    uint16_t* o = p.out + (static_cast<int64_t>(s.start + i) * p.NKV + h) * p.G * D + g * D + col;
    *reinterpret_cast<uint32_t*>(o) = Ops<T>::pack(x * inv, y * inv);
  }
}

// ---- host ---------------------------------------------------------------------------------------

bool bad_ptr(const void* p, uintptr_t mask) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) & mask) != 0;
}

// Workgroups that a CU holds, and that the list is cut for (more of them would wait for a place and begin
// anew): by their LDS two, and one of heads over 128.
int held(int32_t D) { return D > 128 ? 1 : 2; }
// Bytes of keys and values that the block tables can hold from which they are read past the caches: what the
// Infinity Cache (256 MB, other tensors in it too) does not keep for a next call.  MI355X, past / through the caches:
// 64 sequences of up to 8192 keys, 8 heads of 128 (1 GB) 176 / 195 us; 14 of up to 4096, 4 of 256 (224 MB) 32.9 / 35.5;
// 12 of 4096, 16 of 64 (192 MB) 26.0 / 26.9; 10 of them (160 MB) 23.0 / 22.8; 8 (128 MB) 19.4 / 19.3; 16 of 4096, 4 of 96
// (96 MB) 18.0 / 17.3.  Not where several row tiles of a sequence read the same keys (16 sequences' 16 tokens of 32
// heads over 8192 keys 126 instead of 118).  What the lengths hold of a table is known to the device alone: short
// sequences in wide tables are read past the caches too.
constexpr int64_t kPastFrom = int64_t{176} << 20;
constexpr int64_t kMostKeys = int64_t{1} << 30;

// Row blocks of 16 a tile: what a sequence's rows fill on average, two at most.  (Four, whose sums leave a CU one
// workgroup, with one product of the weights: 8 sequences of up to 4096 keys with 54 rows 22.0 us instead of 18.4, 2 x
// 512 tokens of 12 heads over 2048 keys 59 / 49, 8 x 64 of 32 heads over 4096 78 / 83.)
int blocks_of(int64_t rows, int32_t B, int32_t G) { return B > 0 && rows * G > int64_t{16} * B ? 2 : 1; }

struct Plan {
  int nb, parts, parts_of_item;
  bool join, many, tiled;     // something to join; of many items; of several of a sequence's rows
  int64_t first_bytes, bytes;
};

// false: more chunks than 32 bits count.
bool plan_of(int64_t rows, int32_t B, int32_t G, int32_t NKV, int32_t D, int64_t most_keys, Plan& pl) {
  pl.nb = blocks_of(rows, B, G);
  const int R = 16 * pl.nb;
  const int64_t chunks = std::max<int64_t>((most_keys + kChunk - 1) / kChunk, 1);
  const int64_t items = (rows * G / R + B) * NKV;
  if (items > 0 && chunks > ((int64_t{1} << 31) - 1) / items) return false;
  const int64_t list = items * chunks + items;      // (each item's rounding included)
  pl.parts = static_cast<int>(std::max<int64_t>(std::min<int64_t>(list, int64_t{held(D)} * device_cu_count()), 1));
  pl.join = chunks > 1;
  pl.tiled = rows * G > int64_t{R} * B;
  pl.many = 2 * items > pl.parts;
  pl.parts_of_item = static_cast<int>(std::min<int64_t>(pl.parts / std::max<int64_t>(items, 1), chunks));
  pl.first_bytes = (4 * (int64_t{B} + 3) + 15) / 16 * 16;
  pl.bytes = pl.first_bytes + 2 * int64_t{pl.parts} * R * (D + 2) * 4;
  return true;
}

template <typename T, int DP>
int launch_paged(const PagedArgs& a, const Plan& pl, hipStream_t s) {
  const bool past = !pl.tiled && a.max_pages * a.page_size * a.B > kPastFrom / (int64_t{4} * a.NKV * a.D);
  const dim3 grid(pl.parts), block(kThreads);
  auto run = [&](auto nb) -> int {
    constexpr int NB = decltype(nb)::value;
    const int rc = past ? launch_kernel(paged_attention_kernel<T, DP, NB, true>, grid, block, s, a)
                        : launch_kernel(paged_attention_kernel<T, DP, NB, false>, grid, block, s, a);
    if (rc != kOk || !pl.join) return rc;
    if (pl.many) return launch_kernel(paged_join_last_kernel<T, 16 * NB>, grid, block, s, a);
    const dim3 join(static_cast<unsigned>(a.rows * a.NKV * a.G), static_cast<unsigned>((a.D + kJoinCols - 1) / kJoinCols));
    // (by the parts that a row can have, when every item is one of equals)
    if (pl.parts_of_item > 64) return launch_kernel(paged_join_kernel<T, 16 * NB, 1024>, join, dim3(1024), s, a);
    if (pl.parts_of_item > 8) return launch_kernel(paged_join_kernel<T, 16 * NB, 256>, join, dim3(256), s, a);
    return launch_kernel(paged_join_kernel<T, 16 * NB, 64>, join, dim3(64), s, a);
  };
  using std::integral_constant;
  if (pl.nb == 1) return run(integral_constant<int, 1>{});
  return run(integral_constant<int, 2>{});
}

}  // namespace
}  // namespace soupk

using namespace soupk;

extern "C" __attribute__((visibility("default"))) int soupk_paged_attention_workspace(
    int64_t rows, int32_t B, int32_t NH, int32_t NKV, int32_t D, int64_t max_pages, int32_t page_size,
    int64_t* bytes) {
  Plan pl;
  if (bytes == nullptr || rows < 0 || B < 0 || NKV < 1 || NH < NKV || NH % NKV || D < 16 || D % 16 || D > 256 ||
      page_size < 1 || max_pages < 0 || max_pages > kMostKeys / page_size ||
      !plan_of(rows, B, NH / NKV, NKV, D, max_pages * page_size, pl))
    return kInvalid;
  *bytes = pl.bytes;
  return kOk;
}

extern "C" __attribute__((visibility("default"))) int soupk_paged_attention(
    const void* q, int64_t q_stride, const void* k_pages, const void* v_pages, int64_t n_pages,
    int64_t page_stride, int32_t page_size, const int32_t* block_table, int64_t max_pages,
    const int32_t* lengths, const int32_t* cu, int32_t B, void* out, int32_t dtype, int64_t rows, int32_t NH,
    int32_t NKV, int32_t D, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  Plan pl;
  if (rows < 0 || B < 0 || NKV < 1 || NH < NKV || NH > (1 << 16) || NH % NKV || D < 16 || D % 16 || D > 256 ||
      page_size < 1 || n_pages < 1 || n_pages >= (int64_t{1} << 31) || max_pages < 0 ||
      max_pages > kMostKeys / page_size || q_stride < 0 ||
      (n_pages > 1 && (page_stride < static_cast<int64_t>(NKV) * page_size * D || page_stride % 8)) ||
      rows > kMaxGrid / NH || (cu == nullptr && rows != B) ||
      !(scale >= -1e30f && scale <= 1e30f) ||
      (dtype != SOUPK_DTYPE_F16 && dtype != SOUPK_DTYPE_BF16) ||
      !plan_of(rows, B, NH / NKV, NKV, D, max_pages * page_size, pl))
    return kInvalid;
  if (rows == 0) return kOk;
  if (bad_elem_ptr(q, dtype) || bad_ptr(out, 3) || bad_ptr(workspace, 15) || workspace_bytes < pl.bytes)
    return kInvalid;
  if (B < 1 || bad_ptr(lengths, 3) || (cu != nullptr && bad_ptr(cu, 3))) return kInvalid;
  if (max_pages > 0 && bad_ptr(block_table, 3)) return kInvalid;
  if (bad_ptr(k_pages, 15) || bad_ptr(v_pages, 15)) return kInvalid;
  PagedArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_pages),
              static_cast<const uint16_t*>(v_pages), block_table, lengths, cu, static_cast<uint16_t*>(out),
              static_cast<uint32_t*>(workspace),
              reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.first_bytes), rows, q_stride,
              max_pages, n_pages, page_stride, B, NKV, NH / NKV, D, page_size, pl.parts,
              static_cast<int>(max_pages * page_size), pl.tiled, scale * kLog2e,
              FastDiv(static_cast<uint32_t>(page_size)), FastDiv(static_cast<uint32_t>(NH / NKV)),
              FastDiv(static_cast<uint32_t>(D / 4))};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto tag) -> int {
    using E = typename decltype(tag)::type;
    if constexpr (std::is_same_v<E, float>) {
      return kInvalid;
    } else {
      if (D <= 64) return launch_paged<E, 64>(a, pl, s);
      if (D <= 96) return launch_paged<E, 96>(a, pl, s);
      if (D <= 128) return launch_paged<E, 128>(a, pl, s);
      return launch_paged<E, 256>(a, pl, s);
    }
  });
}
