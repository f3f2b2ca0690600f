// Rotary positions for any part of a head, in either layout: the tables of cosines and sines (scaled
// for long contexts), the rotation with its gradient, and the append of new tokens' keys and values to a
// paged cache with the rotation applied on the way.
//
// Tables: pair i of dim / 2 turns by inv_i = theta^(-2 i / dim) a position; cos, sin of t * inv_i, times
// a gain.  Scalings (frequencies in 64 bits on the host, passed by value):
//   linear   inv_i / factor
//   dynamic  theta' = theta (factor n / n0 - (factor - 1))^(dim / (dim - 2)) once n = seq exceeds the
//            original length n0 (the "NTK-aware" base)
//   yarn     (Peng et al. 2023, "YaRN: Efficient Context Window Extension of Large Language Models")
//            inv_i (1 - r_i) + inv_i / factor * r_i, with a ramp r_i over the pair's number from the pair
//            that turns beta_fast times within n0 to the one that turns beta_slow times; the gain is
//            0.1 ln(factor) + 1
// An angle is held in turns, as two 64-bit numbers, and reduced to the nearest quarter before its cosine and
// sine are summed from their Taylor series, which end 2e-10 early: at position 2^20 an angle in fp32 would be 0.03
// rad off.  A frequency made from theta is rounded to 64 bits (1e-15 of the angle, 1e-9 rad at 10^6 rad);
// a given one is taken exactly.
//
// Rotation: (a, b) -> (a c - b s, b c + a s) for the pairs (x[i], x[i + R/2]) or, interleaved,
// (x[2 i], x[2 i + 1]) of the leading R = dim elements of a head; the others are copied.  Products and
// sums are rounded one at a time in fp32, as in the padded and token-major rotations of this library, so
// that a token appended to the cache has the bits that the training path gives it.  The gradient is the same
// with -s.
//
// What bounds them is memory: MI355X, the rotation of 8192 tokens of 40 heads of 128 in bf16, half of each
// interleaved, 29 us each way (5.9 TB/s); 8192 tokens of 48 heads appended 33 us (5.4 TB/s); tables of 131072
// positions of 128 12.2 us (67 MB of stores; the angles hide behind them).  A few tokens are bound by the host.
//
// Mapping: an item is 16 elements of a head, two runs of 8 (by halves they rotate against each other); a
// wavefront takes the items of 64 / (D / 16) neighbouring heads of one token, PER times over, so that one read
// of the token's table row serves PER heads.  A head that cannot be cut so (D or the rotated part no multiple
// of 16) takes a pair per lane instead.

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "elem.hpp"
#include "fastdiv.hpp"

namespace soupk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

// ---- tables -------------------------------------------------------------------------------------

constexpr int kMaxPairs = 128;
// Positions of a thread where there are many, whose first sum serves the others: 131072 positions of 128 in 15.0
// us with one, 15.4 with two, 12.4 with four, 12.2 with eight (12.1 with nothing but the stores); 4096 positions
// 6.9 -> 6.5.
constexpr int kPositions = 8;
constexpr int64_t kManyThreads = 16384;
struct Turns {                    // a position's part of a turn: a double, and what that left
  double per_pos[kMaxPairs], rest[kMaxPairs];
};
// Position `pos`'s turns of frequency f + rest, whole ones taken off.  (The product's rounding is added back: at 10^13
// rad it is 10^-3 rad.)
__device__ __forceinline__ double turns_at(double pos, double f, double rest) {
  const double t = pos * f;
  return t - __builtin_rint(t) + __builtin_fma(pos, rest, __builtin_fma(pos, f, -t));
}

// cos and sin of 2 pi r for r in [-1/2, 1/2]: quarter turns split off, then the series of the remaining
// |x| <= pi / 4 (first terms left out: x^13 / 13! < 7e-12, x^12 / 12! < 2e-10; an fp32 number near 1 is
// rounded by up to 3e-8).
__device__ __forceinline__ void cos_sin_turns(double r, double& c, double& s) {
  const double q = __builtin_rint(4.0 * r);
  const double x = __builtin_fma(q, -0.25, r) * 6.283185307179586476925;
  const double y = x * x;
  double sn = -1.0 / 39916800.0;
  sn = __builtin_fma(sn, y, 1.0 / 362880.0);
  sn = __builtin_fma(sn, y, -1.0 / 5040.0);
  sn = __builtin_fma(sn, y, 1.0 / 120.0);
  sn = __builtin_fma(sn, y, -1.0 / 6.0);
  sn = __builtin_fma(sn * y, x, x);
  double cs = -1.0 / 3628800.0;
  cs = __builtin_fma(cs, y, 1.0 / 40320.0);
  cs = __builtin_fma(cs, y, -1.0 / 720.0);
  cs = __builtin_fma(cs, y, 1.0 / 24.0);
  cs = __builtin_fma(cs, y, -0.5);
  cs = __builtin_fma(cs, y, 1.0);
  const int quarter = static_cast<int>(q) & 3;
  const double a = quarter & 1 ? sn : cs, b = quarter & 1 ? cs : sn;
  c = quarter == 1 || quarter == 2 ? -a : a;
  s = quarter >= 2 ? -b : b;
}

// N pairs of every `step`-th position a thread, P of them: the first angle's cosine and sine are summed, and
// turned on by the step's (each turn rounds 1e-16) to the next ones.
template <int N, int P>
__global__ __launch_bounds__(kThreads) void rotary_tables_kernel(Turns turns, float* __restrict__ cos_t,
                                                                 float* __restrict__ sin_t, double gain,
                                                                 uint32_t step, uint32_t seq,
                                                                 FastDiv per_pos, int half) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t q = per_pos.div(i), g = i - q * per_pos.d;
  // (positions in blocks of P * step, a thread's `step` apart)
  const uint32_t first = P == 1 ? q : q / step * (P * step) + q % step;
  if (first >= seq) return;
  double c[N], s[N], cs[N], ss[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const double f = turns.per_pos[g * N + j], rest = turns.rest[g * N + j];
    cos_sin_turns(turns_at(first, f, rest), c[j], s[j]);
    c[j] *= gain;
    s[j] *= gain;
    if constexpr (P > 1) {
      cos_sin_turns(turns_at(step, f, rest), cs[j], ss[j]);
    }
  }
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const uint32_t pos = first + k * step;
    if (P > 1 && pos >= seq) return;
    const int64_t at = static_cast<int64_t>(pos) * half + g * N;
    if constexpr (N == 4) {
      f32x4 a, b;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        a[j] = static_cast<float>(c[j]);
        b[j] = static_cast<float>(s[j]);
      }
      *reinterpret_cast<f32x4*>(cos_t + at) = a;
      *reinterpret_cast<f32x4*>(sin_t + at) = b;
    } else {
      cos_t[at] = static_cast<float>(c[0]);
      sin_t[at] = static_cast<float>(s[0]);
    }
    if (k + 1 < P) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const double x = __builtin_fma(c[j], cs[j], -(s[j] * ss[j]));
        s[j] = __builtin_fma(s[j], cs[j], c[j] * ss[j]);
        c[j] = x;
      }
    }
  }
}

// ---- the rotation of an item --------------------------------------------------------------------

// What part of a head an item covers: N elements from `a` and N from `b` (in elements of the head); the first
// pairs of both in the tables, or -1 where a run's elements are copied.
struct Item {
  int a, b, turn_a, turn_b;
  bool two;           // (N = 1) there is a second element
};

struct Layout {
  int D, half;        // head dim; rotated pairs (R / 2)
  int items;          // of a head
  bool interleaved;
};

// (Neighbouring items are neighbours in memory, run by run, so that a wavefront's access covers whole lines
// where it can.  Interleaved pairs lie within a run, and the runs of an item are the same place of both halves
// of the head; as 16 neighbouring elements an access touched every other 16 bytes: 8192 tokens of 40
// heads, half of each rotated, both ways 74 us instead of 57.)
template <int N>
__device__ __forceinline__ Item item_of(const Layout& l, int i) {
  if constexpr (N > 1) {
    if (l.interleaved) {
      const int a = N * i, b = l.D / 2 + N * i;
      return {a, b, a < 2 * l.half ? a / 2 : -1, b < 2 * l.half ? b / 2 : -1, true};
    }
  }
  const int turned = l.half / N;
  if (i < turned) {
    if (N == 1 && l.interleaved) return {2 * i, 2 * i + 1, i, i, true};
    return {N * i, l.half + N * i, N * i, N * i, true};
  }
  const int at = 2 * l.half + N * (i - turned), next = at + N * (l.items - turned);
  return {at, next, -1, -1, next < l.D};
}

// x, y: the item's two runs, c, s: the cosines and sines of their pairs (interleaved: of x's N / 2, then of
// y's).
template <int N>
__device__ __forceinline__ void turn(float (&x)[N], float (&y)[N], const float (&c)[N], const float (&s)[N],
                                     const Item& it, bool interleaved) {
  if (N > 1 && interleaved) {
    auto pairs = [&](float (&v)[N], int first) {
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        const int u = first + j / 2;
        const float a = v[j] * c[u] - v[j + 1] * s[u], b = v[j + 1] * c[u] + v[j] * s[u];
        v[j] = a;
        v[j + 1] = b;
      }
    };
    if (it.turn_a >= 0) pairs(x, 0);
    if (it.turn_b >= 0) pairs(y, N / 2);
  } else if (it.turn_a >= 0) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float a = x[j] * c[j] - y[j] * s[j], b = y[j] * c[j] + x[j] * s[j];
      x[j] = a;
      y[j] = b;
    }
  }
}

template <typename T, int N, bool NT>
__device__ __forceinline__ void load_run(const char* base, int64_t at, float (&v)[N]) {
  if constexpr (N == 8)
    Elem<T>::unpack8(Elem<T>::template load8<NT>(base + at * Elem<T>::kBytes), v);
  else
    v[0] = Elem<T>::load1(base + at * Elem<T>::kBytes);
}
template <typename T, int N, bool NT>
__device__ __forceinline__ void store_run(char* base, int64_t at, const float (&v)[N]) {
  if constexpr (N == 8)
    Elem<T>::template store8<NT>(base + at * Elem<T>::kBytes, v);
  else
    Elem<T>::store1(base + at * Elem<T>::kBytes, v[0]);
}

// The cosines and (times `sign`) sines of an item's pairs, in the order of turn(); nothing for a run that is
// copied.
template <int N>
__device__ __forceinline__ void load_turns(const float* cos_t, const float* sin_t, int64_t row, const Item& it,
                                           float sign, bool interleaved, float (&c)[N], float (&s)[N]) {
  if constexpr (N == 8) {
    const int second = interleaved ? it.turn_b : it.turn_a >= 0 ? it.turn_a + 4 : -1;
    if (it.turn_a >= 0) {
      load_n<float, 4, false>(reinterpret_cast<const char*>(cos_t + row + it.turn_a), c);
      load_n<float, 4, false>(reinterpret_cast<const char*>(sin_t + row + it.turn_a), s);
    }
    if (second >= 0) {
      load_n<float, 4, false>(reinterpret_cast<const char*>(cos_t + row + second), c + 4);
      load_n<float, 4, false>(reinterpret_cast<const char*>(sin_t + row + second), s + 4);
    }
  } else if (it.turn_a >= 0) {
    c[0] = cos_t[row + it.turn_a];
    s[0] = sin_t[row + it.turn_a];
  }
#pragma unroll
  for (int j = 0; j < N; ++j) s[j] = s[j] * sign;
}

// ---- the rotation -------------------------------------------------------------------------------

struct RotaryArgs {
  const char* x;
  const float* cos_t;
  const float* sin_t;
  const int64_t* pos;
  char* out;
  int64_t n_pos, table_stride, row_stride, head_stride;
  int heads;              // of a token
  FastDiv per_tok;        // divides by the wavefront items of a token
  Layout l;
  float sign;
};

// A wavefront takes PER * slots neighbouring heads of one token, slots = 64 / items.
template <typename T, int N, int PER>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs p, int64_t row0, uint32_t waves) {
  const uint32_t wi = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (wi >= waves) return;
  const uint32_t tok = p.per_tok.div(wi);
  const int group = static_cast<int>(wi - tok * p.per_tok.d);
  const int64_t row = row0 + tok;
  const int lane = threadIdx.x & 63;
  const int slots = max(kWave / p.l.items, 1);
  const int64_t t = p.pos[row];
  const bool placed = t >= 0 && t < p.n_pos;
  // (more than 64 items a head, in pairs: a lane takes every 64th)
  for (int i0 = lane % (slots == 1 ? kWave : p.l.items); i0 < p.l.items; i0 += kWave) {
    const int slot = slots == 1 ? 0 : lane / p.l.items;
    if (slot >= slots) break;
    const Item it = item_of<N>(p.l, i0);
    float c[N], s[N], x[PER][N], y[PER][N];
    const int h0 = group * PER * slots + slot;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      // (heads too many read the last one again)
      const int64_t at = row * p.row_stride + min(h0 + u * slots, p.heads - 1) * p.head_stride;
      load_run<T, N, true>(p.x, at + it.a, x[u]);
      if (N > 1 || it.two) load_run<T, N, true>(p.x, at + it.b, y[u]);
    }
    if (placed) load_turns<N>(p.cos_t, p.sin_t, t * p.table_stride, it, p.sign, p.l.interleaved, c, s);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int h = h0 + u * slots;
      if (h >= p.heads) break;
      if (!placed) {
#pragma unroll
        for (int j = 0; j < N; ++j) x[u][j] = y[u][j] = 0.f;
      } else {
        turn<N>(x[u], y[u], c, s, it, p.l.interleaved);
      }
      const int64_t at = (row * p.heads + h) * p.l.D;
      store_run<T, N, true>(p.out, at + it.a, x[u]);
      if (N > 1 || it.two) store_run<T, N, true>(p.out, at + it.b, y[u]);
    }
  }
}

// The same with one run of N elements a lane, in the order of memory; by halves, a run's partner is in another
// lane of its head.  Every access covers whole lines, where runs of R / 2 elements would not be ones.
template <typename T, int N, bool NT>
__device__ __forceinline__ void load_some(const char* base, int64_t at, float (&v)[N]) {
  const char* p = base + at * Elem<T>::kBytes;
  if constexpr (N >= 4) {
    load_n<T, N, NT>(p, v);
  } else {
    static_assert(N == 2, "");
    v[0] = Elem<T>::load1(p);
    v[1] = Elem<T>::load1(p + Elem<T>::kBytes);
  }
}
template <typename T, int N, bool NT>
__device__ __forceinline__ void store_some(char* base, int64_t at, const float (&v)[N]) {
  char* p = base + at * Elem<T>::kBytes;
  if constexpr (N >= 4) {
    store_n<T, N, NT>(p, v);
  } else if constexpr (std::is_same_v<T, float>) {
    *reinterpret_cast<float*>(p) = v[0];
    *reinterpret_cast<float*>(p + 4) = v[1];
  } else {
    typedef uint32_t word __attribute__((aligned(2)));
    *reinterpret_cast<word*>(p) = std::is_same_v<T, f16> ? pack_h2(v[0], v[1]) : pack_b2(v[0], v[1]);
  }
}

template <typename T, int N, int PER>
__global__ __launch_bounds__(kThreads) void rotary_lines_kernel(RotaryArgs p, int64_t row0, uint32_t waves) {
  const uint32_t wi = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (wi >= waves) return;
  const uint32_t tok = p.per_tok.div(wi);
  const int group = static_cast<int>(wi - tok * p.per_tok.d);
  const int64_t row = row0 + tok;
  const int lane = threadIdx.x & 63, items = p.l.items, slots = kWave / items;
  const int64_t t = p.pos[row];
  const bool placed = t >= 0 && t < p.n_pos;
  // (lanes too many repeat the last head's)
  const int slot = min(lane / items, slots - 1), i = lane - lane / items * items;
  const int a = N * i, h0 = group * PER * slots + slot;
  const bool turned = a < 2 * p.l.half && placed, second = a >= p.l.half;
  float x[PER][N], c[N], s[N];
#pragma unroll
  for (int u = 0; u < PER; ++u)
    load_some<T, N, true>(p.x, row * p.row_stride + min(h0 + u * slots, p.heads - 1) * p.head_stride + a, x[u]);
  if (turned) {
    if (p.l.interleaved) {
      const int64_t at = t * p.table_stride + a / 2;
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        c[j] = p.cos_t[at + j];
        s[j] = p.sin_t[at + j] * p.sign;
      }
    } else {
      const int64_t at = t * p.table_stride + (second ? a - p.l.half : a);
      load_some<float, N, false>(reinterpret_cast<const char*>(p.cos_t), at, c);
      load_some<float, N, false>(reinterpret_cast<const char*>(p.sin_t), at, s);
#pragma unroll
      for (int j = 0; j < N; ++j) s[j] = s[j] * (second ? p.sign : -p.sign);
    }
  }
  const int partner = lane + (second ? -1 : 1) * (p.l.half / N);
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    float y[N];
    if (!p.l.interleaved) {
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = __shfl(x[u][j], partner);
    }
    if (!placed) {
#pragma unroll
      for (int j = 0; j < N; ++j) x[u][j] = 0.f;
    } else if (turned) {
      if (p.l.interleaved) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
          const float v = x[u][j] * c[j / 2] - x[u][j + 1] * s[j / 2];
          x[u][j + 1] = x[u][j + 1] * c[j / 2] + x[u][j] * s[j / 2];
          x[u][j] = v;
        }
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[u][j] = x[u][j] * c[j] + y[j] * s[j];
      }
    }
    const int h = h0 + u * slots;
    if (h < p.heads && lane < slots * items)
      store_some<T, N, true>(p.out, (row * p.heads + h) * p.l.D + a, x[u]);
  }
}

// ---- append to a paged cache --------------------------------------------------------------------

struct AppendArgs {
  const char* qkv;
  const char* lora_q;
  const char* lora_v;
  const float* cos_t;       // null: no rotation
  const float* sin_t;
  const int32_t* cu;        // null: one new token a sequence
  const int32_t* lengths;
  const int32_t* table;
  char* q_out;
  char* k_pages;
  char* v_pages;
  int64_t n_pos, table_stride, pages, max_pages, page_stride, rows;
  int32_t B;
  int NH, NKV;
  bool lora_f32;
  FastDiv per_tok, per_page;      // by the wavefront items of a token, by a page's slots
  Layout l;
};

// The sequence that token `tok` belongs to (the last one that starts at or before it; -1: none), found 64
// bounds at a time, and its bounds.  All lanes of the wavefront together.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int32_t B, int64_t tok, int64_t rows,
                                           int64_t& start, int64_t& end) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = B + 1;
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave;
    const int at = lo + lane * step;
    const bool below = lane * step < n && at <= B && cu[at] <= tok;
    const int count = __popcll(__ballot(below));
    if (count == 0) return -1;
    lo += (count - 1) * step;
    n = min(step, B + 1 - lo);
    if (step == 1) break;
  }
  if (lo >= B) return -1;
  start = cu[lo];
  end = cu[lo + 1];
  return start >= 0 && start <= tok && tok < end && end <= rows ? lo : -1;
}

template <typename T, int N, int PER>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(AppendArgs p, int64_t row0, uint32_t waves) {
  const uint32_t wi = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (wi >= waves) return;
  const uint32_t tok = p.per_tok.div(wi);
  const int group = static_cast<int>(wi - tok * p.per_tok.d);
  const int64_t row = row0 + tok;
  const int lane = threadIdx.x & 63;
  const int heads = p.NH + 2 * p.NKV, D = p.l.D;
  const int slots = max(kWave / p.l.items, 1);
  // the token's place: sequence, position, page and slot
  int64_t t = -1, base = 0;
  bool placed = false;
  int64_t start = row, end = row + 1;
  const int b = p.cu != nullptr ? sequence_of(p.cu, p.B, row, p.rows, start, end)
                                : (row < p.B ? static_cast<int>(row) : -1);
  if (b >= 0) {
    t = p.lengths[b] - end + row;
    if (t >= 0 && (p.cos_t == nullptr || t < p.n_pos)) {
      const uint32_t pg = p.per_page.div(static_cast<uint32_t>(t));
      if (pg < p.max_pages) {
        const int64_t page = p.table[b * p.max_pages + pg];
        placed = page >= 0 && page < p.pages;
        base = page * p.page_stride + (t - static_cast<int64_t>(pg) * p.per_page.d) * D;
      }
    }
  }
  for (int i0 = lane % (slots == 1 ? kWave : p.l.items); i0 < p.l.items; i0 += kWave) {
    const int slot = slots == 1 ? 0 : lane / p.l.items;
    if (slot >= slots) break;
    const Item it = item_of<N>(p.l, i0);
    float c[N], s[N], x[PER][N], y[PER][N];
    const int h0 = group * PER * slots + slot;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int64_t at = (row * heads + min(h0 + u * slots, heads - 1)) * D;
      load_run<T, N, true>(p.qkv, at + it.a, x[u]);
      if (N > 1 || it.two) load_run<T, N, true>(p.qkv, at + it.b, y[u]);
    }
    if (placed && p.cos_t != nullptr)
      load_turns<N>(p.cos_t, p.sin_t, t * p.table_stride, it, 1.f, p.l.interleaved, c, s);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int h = h0 + u * slots;
      if (h >= heads) break;
      const bool is_q = h < p.NH, is_v = h >= p.NH + p.NKV;
      if (!placed) {
        if (!is_q) continue;
#pragma unroll
        for (int j = 0; j < N; ++j) x[u][j] = y[u][j] = 0.f;
      } else {
        const char* lora = is_q ? p.lora_q : is_v ? p.lora_v : nullptr;
        if (lora != nullptr) {
          const int64_t at = is_q ? (row * p.NH + h) * D : (row * p.NKV + (h - p.NH - p.NKV)) * D;
          float dx[N], dy[N];
          if (p.lora_f32) {
            load_run<float, N, true>(lora, at + it.a, dx);
            if (N > 1 || it.two) load_run<float, N, true>(lora, at + it.b, dy);
          } else {
            load_run<T, N, true>(lora, at + it.a, dx);
            if (N > 1 || it.two) load_run<T, N, true>(lora, at + it.b, dy);
          }
#pragma unroll
          for (int j = 0; j < N; ++j) {
            x[u][j] = x[u][j] + dx[j];
            if (N > 1 || it.two) y[u][j] = y[u][j] + dy[j];
          }
        }
        if (!is_v && p.cos_t != nullptr) turn<N>(x[u], y[u], c, s, it, p.l.interleaved);
      }
      if (is_q) {
        const int64_t at = (row * p.NH + h) * D;
        store_run<T, N, false>(p.q_out, at + it.a, x[u]);
        if (N > 1 || it.two) store_run<T, N, false>(p.q_out, at + it.b, y[u]);
      } else {
        char* pages = is_v ? p.v_pages : p.k_pages;
        const int64_t at = base + static_cast<int64_t>(is_v ? h - p.NH - p.NKV : h - p.NH) * p.per_page.d * D;
        store_run<T, N, false>(pages, at + it.a, x[u]);
        if (N > 1 || it.two) store_run<T, N, false>(pages, at + it.b, y[u]);
      }
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------

bool bad_ptr(const void* p, uintptr_t mask) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) & mask) != 0;
}

// Whether a head is cut into items of two runs of 8, and its items.
bool in_runs(Layout& l) {
  const int R = 2 * l.half;
  const bool runs = l.D % 16 == 0 && R % 16 == 0 && l.D <= 16 * kWave;
  l.items = runs ? l.D / 16 : l.half + (l.D - R + 1) / 2;
  return runs;
}

constexpr int64_t kMostWaves = kMaxGrid * kWaves;     // of one launch

// Launches `run(args, first row, wavefronts)` over all rows; set(per): wavefront items of a token.
template <class F>
int over_rows(int64_t rows, int64_t per_tok, F&& run) {
  const int64_t step = std::max<int64_t>(1, std::min<int64_t>(kMostWaves, (int64_t{1} << 31) - 1) / per_tok);
  for (int64_t r = 0; r < rows; r += step) {
    const int64_t waves = std::min(step, rows - r) * per_tok;
    const int rc = run(r, static_cast<uint32_t>(waves),
                       dim3(static_cast<unsigned>((waves + kWaves - 1) / kWaves)));
    if (rc != kOk) return rc;
  }
  return kOk;
}

// Wavefront items from which a wavefront takes two groups of heads, or three where they divide a token's (they
// share the token's place and tables), below which one fills the chip sooner.  MI355X: 8192 tokens of 40 heads
// both ways 58.5 us with one, 57.7 with two, 58.4 with three; 8192 tokens of 48 heads appended 36.6, 33.8, 33.1.
constexpr int64_t kTwoFrom = 4096;

// Calls run(tag of <N>, tag of <PER>, groups of a token) for `heads` heads of layout l.
template <class F>
int with_items(Layout& l, int64_t rows, int heads, F&& run) {
  const bool runs = in_runs(l);
  const int slots = std::max(kWave / l.items, 1);
  const int groups = (heads + slots - 1) / slots;
  using std::integral_constant;
  if (!runs) return run(integral_constant<int, 1>{}, integral_constant<int, 1>{}, groups);
  if (rows * groups >= kTwoFrom && groups % 3 == 0)
    return run(integral_constant<int, 8>{}, integral_constant<int, 3>{}, groups / 3);
  if (rows * groups >= kTwoFrom)
    return run(integral_constant<int, 8>{}, integral_constant<int, 2>{}, (groups + 1) / 2);
  return run(integral_constant<int, 8>{}, integral_constant<int, 1>{}, groups);
}

}  // namespace
}  // namespace soupk

using namespace soupk;

extern "C" __attribute__((visibility("default"))) int soupk_rotary_tables(
    float* cos, float* sin, int64_t seq, int32_t dim, const double* inv_freq, double theta, int32_t scaling,
    double factor, double original, double beta_fast, double beta_slow, double gain, void* stream) {
  constexpr double kTwoPi = 6.283185307179586476925;
  if (seq < 0 || seq >= (int64_t{1} << 31) || dim < 2 || dim % 2 || dim > 2 * kMaxPairs) return kInvalid;
  if (!(std::fabs(gain) <= 1e30)) return kInvalid;
  Turns turns;
  const int half = dim / 2;
  auto set = [&](int i, double f) {         // f / (2 pi), of which the second number is below 2^-53 of the first
    constexpr double kPerTurn = 0x1.45f306dc9c883p-3, kLeft = -0x1.6b01ec5417056p-57;
    turns.per_pos[i] = f * kPerTurn;
    turns.rest[i] = std::fma(f, kPerTurn, -turns.per_pos[i]) + f * kLeft;
  };
  if (inv_freq != nullptr) {
    for (int i = 0; i < half; ++i) {
      // (2^31 positions of it are below 2^49 turns, whose parts a double and its rest hold)
      if (!(std::fabs(inv_freq[i]) <= 1e6)) return kInvalid;
      set(i, inv_freq[i]);
    }
  } else {
    if (!(theta > 1.0 && theta <= 1e30)) return kInvalid;
    if (scaling < SOUPK_ROPE_DEFAULT || scaling > SOUPK_ROPE_YARN) return kInvalid;
    if (scaling != SOUPK_ROPE_DEFAULT && !(factor >= 1.0 && factor <= 1e6)) return kInvalid;
    if (scaling >= SOUPK_ROPE_DYNAMIC && !(original >= 1.0 && original <= 2147483648.0)) return kInvalid;
    double low = 0.0, width = 1.0;
    if (scaling == SOUPK_ROPE_DYNAMIC && static_cast<double>(seq) > original && dim > 2)
      theta *= std::pow(factor * static_cast<double>(seq) / original - (factor - 1.0),
                        static_cast<double>(dim) / (dim - 2));
    if (scaling == SOUPK_ROPE_YARN) {
      if (!(beta_slow > 0.0 && beta_fast >= beta_slow && beta_fast <= 1e6)) return kInvalid;
      auto pair = [&](double n) { return dim * std::log(original / (n * kTwoPi)) / (2.0 * std::log(theta)); };
      low = std::fmax(std::floor(pair(beta_fast)), 0.0);
      const double high = std::fmin(std::ceil(pair(beta_slow)), dim - 1.0);
      width = std::fmax(high - low, 0.001);
    }
    const double decay = 2.0 * std::log(theta) / dim;
    for (int i = 0; i < half; ++i) {
      double f = std::exp(-i * decay);
      if (scaling == SOUPK_ROPE_LINEAR) f /= factor;
      if (scaling == SOUPK_ROPE_YARN) {
        const double ramp = std::fmin(std::fmax((i - low) / width, 0.0), 1.0);
        f = f / factor * ramp + f * (1.0 - ramp);
      }
      set(i, f);
    }
  }
  for (int i = half; i < kMaxPairs; ++i) turns.per_pos[i] = turns.rest[i] = 0.0;
  if (seq == 0) return kOk;
  if (bad_ptr(cos, 15) || bad_ptr(sin, 15)) return kInvalid;
  const int n = half % 4 == 0 ? 4 : 1, per = half / n;
  const int ps = seq * per >= kManyThreads ? kPositions : 1;
  const uint32_t step = kThreads / 16;
  const int64_t rows = ps == 1 ? seq : (seq + ps * step - 1) / (ps * step) * step, items = rows * per;
  if (items > kMaxGrid * kThreads - kThreads) return kInvalid;
  auto run = [&](auto kernel) {
    return launch_kernel(kernel, dim3(static_cast<unsigned>((items + kThreads - 1) / kThreads)), dim3(kThreads),
                         static_cast<hipStream_t>(stream), turns, cos, sin, gain, step,
                         static_cast<uint32_t>(seq), FastDiv(static_cast<uint32_t>(per)), half);
  };
  if (ps == 1) return n == 4 ? run(rotary_tables_kernel<4, 1>) : run(rotary_tables_kernel<1, 1>);
  return n == 4 ? run(rotary_tables_kernel<4, kPositions>) : run(rotary_tables_kernel<1, kPositions>);
}

extern "C" __attribute__((visibility("default"))) int soupk_rotary(
    const void* x, int32_t dtype, int64_t row_stride, int64_t head_stride, const float* cos, const float* sin,
    int64_t n_pos, int64_t table_stride, const int64_t* pos, void* out, int64_t rows, int32_t heads, int32_t D,
    int32_t R, int32_t interleaved, int32_t inverse, void* stream) {
  if (rows < 0 || heads < 1 || heads > (1 << 16) || D < 2 || D > (1 << 16) || R < 2 || R % 2 || R > D ||
      n_pos < 0 || row_stride < 0 || head_stride < 0 || table_stride < 0)
    return kInvalid;
  if (dtype != SOUPK_DTYPE_F16 && dtype != SOUPK_DTYPE_BF16 && dtype != SOUPK_DTYPE_F32) return kInvalid;
  if (rows == 0) return kOk;
  if (bad_elem_ptr(x, dtype) || bad_elem_ptr(out, dtype) || bad_ptr(pos, 7) ||
      (n_pos > 0 && (bad_ptr(cos, 3) || bad_ptr(sin, 3))))
    return kInvalid;
  RotaryArgs a{static_cast<const char*>(x), cos, sin, pos, static_cast<char*>(out), n_pos, table_stride,
               row_stride, head_stride, heads, FastDiv(1), Layout{D, R / 2, 0, interleaved != 0},
               inverse ? -1.f : 1.f};
  return with_type(dtype, [&](auto tag) -> int {
    using E = typename decltype(tag)::type;
    auto launch = [&](auto kernel, int groups) {
      a.per_tok = FastDiv(static_cast<uint32_t>(groups));
      return over_rows(rows, groups, [&](int64_t r, uint32_t waves, dim3 grid) {
        return launch_kernel(kernel, grid, dim3(kThreads), static_cast<hipStream_t>(stream), a, r, waves);
      });
    };
    // Runs in the order of memory, of 16 bytes or of two elements; where pairs of runs are whole lines too, in
    // those, which need no exchange.
    constexpr int kBytes = Elem<E>::kBytes, kRun = 16 / kBytes;
    auto in_lines = [&](int n) {
      return D % n == 0 && (interleaved ? R % n == 0 : R / 2 % n == 0) && D / n <= kWave;
    };
    const bool pairs = kBytes == 2 && D % 16 == 0 && D <= 16 * kWave && R % 16 == 0 &&
                       (interleaved ? D / 2 * kBytes % 128 == 0
                                    : R / 2 * kBytes % 128 == 0 && (D - R) / 2 * kBytes % 128 == 0);
    if (!pairs && (in_lines(kRun) || in_lines(2))) {
      const int n = in_lines(kRun) ? kRun : 2;
      a.l.items = D / n;
      const int slots = kWave / a.l.items, groups = (heads + slots - 1) / slots;
      if (n == 2) return launch(rotary_lines_kernel<E, 2, 2>, (groups + 1) / 2);
      if (rows * groups >= kTwoFrom) return launch(rotary_lines_kernel<E, kRun, 2>, (groups + 1) / 2);
      return launch(rotary_lines_kernel<E, kRun, 1>, groups);
    }
    return with_items(a.l, rows, heads, [&](auto n, auto per, int groups) {
      return launch(rotary_kernel<E, decltype(n)::value, decltype(per)::value>, groups);
    });
  });
}

extern "C" __attribute__((visibility("default"))) int soupk_rope_append(
    const void* qkv, const void* lora_q, const void* lora_v, int32_t lora_dtype, const float* cos,
    const float* sin, int64_t n_pos, int64_t table_stride, int32_t R, int32_t interleaved, const int32_t* cu,
    const int32_t* lengths, const int32_t* block_table, int32_t B, int64_t max_pages, void* q_out,
    void* k_pages, void* v_pages, int64_t n_pages, int64_t page_stride, int32_t page_size, int32_t dtype,
    int64_t rows, int32_t NH, int32_t NKV, int32_t D, void* stream) {
  if (rows < 0 || B < 0 || NH < 1 || NH > (1 << 16) || NKV < 1 || NKV > (1 << 16) || D < 16 || D % 16 ||
      D > 256 || page_size < 1 || n_pages < 0 || n_pages >= (int64_t{1} << 31) || max_pages < 0 || n_pos < 0 ||
      table_stride < 0 || max_pages > ((int64_t{1} << 31) - 1) / page_size ||
      (n_pages > 1 && page_stride < static_cast<int64_t>(NKV) * page_size * D))
    return kInvalid;
  if (dtype != SOUPK_DTYPE_F16 && dtype != SOUPK_DTYPE_BF16) return kInvalid;
  const bool rotate = cos != nullptr;
  if (rotate && (R < 2 || R % 2 || R > D)) return kInvalid;
  if ((lora_q || lora_v) && lora_dtype != dtype && lora_dtype != SOUPK_DTYPE_F32) return kInvalid;
  if (rows == 0) return kOk;
  if (bad_elem_ptr(qkv, dtype) || bad_elem_ptr(q_out, dtype) || (rotate && (bad_ptr(cos, 3) || bad_ptr(sin, 3))) ||
      (cu != nullptr && bad_ptr(cu, 3)) || (lora_q && bad_elem_ptr(lora_q, lora_dtype)) ||
      (lora_v && bad_elem_ptr(lora_v, lora_dtype)))
    return kInvalid;
  if (B > 0 && bad_ptr(lengths, 3)) return kInvalid;
  if (B > 0 && max_pages > 0 && bad_ptr(block_table, 3)) return kInvalid;
  if (n_pages > 0 && (bad_elem_ptr(k_pages, dtype) || bad_elem_ptr(v_pages, dtype))) return kInvalid;
  AppendArgs a{static_cast<const char*>(qkv), static_cast<const char*>(lora_q),
               static_cast<const char*>(lora_v), cos, sin, cu, lengths, block_table,
               static_cast<char*>(q_out), static_cast<char*>(k_pages), static_cast<char*>(v_pages), n_pos,
               table_stride, n_pages, max_pages, page_stride, rows, B, NH, NKV,
               lora_dtype == SOUPK_DTYPE_F32, FastDiv(1), FastDiv(static_cast<uint32_t>(page_size)),
               // (without tables every item is copied: cut as if all of the head were rotated)
               Layout{D, rotate ? R / 2 : D / 2, 0, interleaved != 0}};
  return with_type(dtype, [&](auto tag) -> int {
    using E = typename decltype(tag)::type;
    if constexpr (std::is_same_v<E, float>) {
      return kInvalid;
    } else {
      return with_items(a.l, rows, NH + 2 * NKV, [&](auto n, auto per, int groups) {
        a.per_tok = FastDiv(static_cast<uint32_t>(groups));
        return over_rows(rows, groups, [&](int64_t r, uint32_t waves, dim3 grid) {
          return launch_kernel(rope_append_kernel<E, decltype(n)::value, decltype(per)::value>, grid,
                               dim3(kThreads), static_cast<hipStream_t>(stream), a, r, waves);
        });
      });
    }
  });
}
