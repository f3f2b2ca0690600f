// Dropout whose mask is drawn from a counter, in the forward and again in the backward, and never
// stored; optionally added to a residual in the same pass.
//
//   out[r, c] = residual[r, c] + (u(R, c) >= limit ? x[r, c] * scale : 0),   R = rows[r] or r
//   u(R, c)   = word c % 4 of Philox4x32-10 at the counter (c / 4, R, call) under the key `seed`
//
// Philox4x32-10 is the counter-based generator of Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3" (2011): ten rounds of two 32 x 32 -> 64 bit products.  A draw
// depends on its row, column, call and seed alone, not on the number of rows or columns, so tokens
// kept without their padding draw what they draw in the padded layout (`rows` gives the padded
// positions), and the backward, which is the same operation on the gradient, redraws the mask.
// Each element has a 32-bit word of its own: it is dropped with probability limit / 2^32.
//
// The sum with the residual and the product with the scale are rounded in fp32 one after the other
// and once more to the output's type.  A dropped element is replaced, not multiplied by zero, so an
// infinity or NaN under the mask does not survive.
//
// Bound: memory.  On MI355X a copy of 147 MB of fp16 runs at 5.87 TB/s and with the draws at 5.79 (16
// bits per element would give 5.93: the multiplies hide under the traffic, so every element gets the
// full word).  What a thread takes follows the result's type, so that each store of a wavefront fills
// whole lines: 8 columns for 16-bit results, 4 and 4 more 256 items on for fp32 ones.  8192 x 8960 fp16
// into an fp32 residual 128 -> 114 us (6.4 TB/s) against 8 columns in two stores; 16-bit results in 4
// columns take 147 instead of 115 us (forward and backward).

#include <algorithm>
#include <type_traits>

#include "elem.hpp"
#include "fastdiv.hpp"

namespace soupk {
namespace {

constexpr int kDropThreads = 256;

// Columns of an item, and items of a thread: a wavefront's store covers whole lines.  An fp32 result
// goes out as 16 bytes of 4 columns (two items a thread), a 16-bit one as 16 bytes of 8.
template <typename Out>
constexpr int item_cols() {
  return Elem<Out>::kBytes == 4 ? 4 : 8;
}
template <typename Out>
constexpr int thread_items() {
  return Elem<Out>::kBytes == 4 ? 2 : 1;
}

struct Draw {
  uint32_t key0, key1, call0, call1;
  uint32_t limit;     // keep when word >= limit
  bool drop_all;      // limit 2^32
};

__device__ __forceinline__ u32x4 philox(uint32_t block, uint32_t row, const Draw& d) {
  uint32_t c0 = block, c1 = row, c2 = d.call0, c3 = d.call1, k0 = d.key0, k1 = d.key1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * c0;
    const uint64_t b = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c1 = static_cast<uint32_t>(b);
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}

template <typename In, typename Out, bool RES>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(
    const char* __restrict__ x, const char* __restrict__ residual, char* __restrict__ out,
    const int64_t* __restrict__ rows, const int64_t* __restrict__ seed, Draw d, float scale,
    uint32_t items, int64_t row0, int64_t C, FastDiv per_row) {
  constexpr int N = item_cols<Out>(), U = thread_items<Out>();
  if (seed != nullptr) {
    const uint64_t s = static_cast<uint64_t>(*seed);
    d.key0 = static_cast<uint32_t>(s);
    d.key1 = static_cast<uint32_t>(s >> 32);
  }
  const uint32_t i0 = blockIdx.x * (kDropThreads * U) + threadIdx.x;
  float v[U][N], e[U][N];
  uint32_t block[U], drawn[U];
  int64_t at[U];
  int n[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = min(i0 + u * kDropThreads, items - 1);   // (past the end: the last item, unused)
    const uint32_t r = per_row.div(i);
    block[u] = i - r * per_row.d;
    const int64_t row = row0 + r, col = static_cast<int64_t>(block[u]) * N;
    at[u] = row * C + col;
    n[u] = static_cast<int>(min(int64_t{N}, C - col));
    drawn[u] = static_cast<uint32_t>(rows != nullptr ? rows[row] : row);
    if (n[u] == N) {
      load_n<In, N, true>(x + at[u] * Elem<In>::kBytes, v[u]);
      if constexpr (RES) load_n<Out, N, true>(residual + at[u] * Elem<Out>::kBytes, e[u]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        v[u][j] = j < n[u] ? Elem<In>::load1(x + (at[u] + j) * Elem<In>::kBytes) : 0.f;
        if constexpr (RES)
          e[u][j] = j < n[u] ? Elem<Out>::load1(residual + (at[u] + j) * Elem<Out>::kBytes) : 0.f;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
      const u32x4 w = philox(block[u] * (N / 4) + q, drawn[u], d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float& y = v[u][4 * q + j];
        y = (w[j] >= d.limit && !d.drop_all) ? y * scale : 0.f;
        if constexpr (RES) y = e[u][4 * q + j] + y;
      }
    }
    if (i0 + u * kDropThreads >= items) return;
    if (n[u] == N) {
      store_n<Out, N, true>(out + at[u] * Elem<Out>::kBytes, v[u]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n[u]) Elem<Out>::store1(out + (at[u] + j) * Elem<Out>::kBytes, v[u][j]);
    }
  }
}

}  // namespace
}  // namespace soupk

using namespace soupk;

extern "C" __attribute__((visibility("default"))) int soupk_dropout(
    const void* x, int32_t x_dtype, const void* residual, void* out, int32_t out_dtype,
    const int64_t* rows, const int64_t* seed_dev, int64_t seed, int64_t call, int64_t limit,
    float scale, int64_t R, int64_t C, void* stream) {
  if (R < 0 || C < 0 || limit < 0 || limit > (int64_t{1} << 32)) return kInvalid;
  if (C > (int64_t{1} << 32) || (C > 0 && R > (int64_t{1} << 62) / C)) return kInvalid;
  if (x_dtype != out_dtype && x_dtype != SOUPK_DTYPE_F32 && out_dtype != SOUPK_DTYPE_F32)
    return kInvalid;
  if (R == 0 || C == 0) return kOk;
  if (bad_elem_ptr(x, x_dtype) || bad_elem_ptr(out, out_dtype)) return kInvalid;
  if (residual != nullptr && bad_elem_ptr(residual, out_dtype)) return kInvalid;
  if ((reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(seed_dev)) & 7u)
    return kInvalid;
  const uint64_t key = static_cast<uint64_t>(seed), off = static_cast<uint64_t>(call);
  const bool all = limit == (int64_t{1} << 32);
  const Draw d{static_cast<uint32_t>(key), static_cast<uint32_t>(key >> 32),
               static_cast<uint32_t>(off), static_cast<uint32_t>(off >> 32),
               all ? 0xffffffffu : static_cast<uint32_t>(limit), all};
  return with_type(x_dtype, [&](auto in) {
    return with_type(out_dtype, [&](auto o) -> int {
      using In = typename decltype(in)::type;
      using Out = typename decltype(o)::type;
      if constexpr (std::is_same_v<In, Out> || std::is_same_v<In, float> ||
                    std::is_same_v<Out, float>) {
        constexpr int64_t kCols = item_cols<Out>(), kPer = kDropThreads * thread_items<Out>();
        const int64_t per_row = (C + kCols - 1) / kCols;      // (<= 2^30: a row fits one launch)
        const int64_t rows_per = std::max<int64_t>(1, ((int64_t{1} << 31) - 1 - kPer) / per_row);
        const FastDiv div(static_cast<uint32_t>(per_row));
        for (int64_t r0 = 0; r0 < R; r0 += rows_per) {
          const uint32_t items = static_cast<uint32_t>(std::min(rows_per, R - r0) * per_row);
          const dim3 grid(static_cast<unsigned>((items + kPer - 1) / kPer)), block(kDropThreads);
          hipStream_t s = static_cast<hipStream_t>(stream);
          auto run = [&](auto kernel) {
            return launch_kernel(kernel, grid, block, s, static_cast<const char*>(x),
                                 static_cast<const char*>(residual), static_cast<char*>(out),
                                 rows, seed_dev, d, scale, items, r0, C, div);
          };
          const int rc = residual != nullptr ? run(dropout_kernel<In, Out, true>)
                                             : run(dropout_kernel<In, Out, false>);
          if (rc != kOk) return rc;
        }
        return kOk;
      } else {
        return kInvalid;
      }
    });
  });
}
