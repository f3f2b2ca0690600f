// RMS norm of every query and key head with the position rotation in the same pass, into the
// token-major q|k|v rows that the varlen attention reads, and its backward.
//
// Per token and query or key head of D dims (the two halves of a head rotate against each other):
//   x = qkv (+ lora_q for a query head), r = 1 / sqrt(mean(x^2) + eps), n = x * r, y = n * w
//   out1 = y1 c1 - y2 s1, out2 = y2 c2 + y1 s2;   a value head passes through (+ lora_v)
// Backward, with g the gradient of out:
//   gy1 = g1 c1 + g2 s2, gy2 = g2 c2 - g1 s1;  dw = sum over tokens and heads of gy * n
//   dx = r * (gy w - n * mean(gy w n));        a value head's gradient passes through
// All in fp32 with fused multiply-adds, one rounding to the rows' type at the store; x and r are formed
// again in the backward from the rows it has to read anyway, so nothing is kept of the forward.
//
// Mapping (forward): a head is a group of G = 2^k lanes, each with 8 dims of the first half and the 8 dims of
// the second half they rotate with, so the rotation is inside a lane and the mean of squares one
// DPP reduction of at most 16 lanes.  A wavefront takes 64 / G neighbouring heads of one token (8
// at D = 128: its loads and stores are whole rows of 2 KiB), or two such groups, which share the
// token's cos / sin.  Those and the weight come from the caches.
//
// The weights' gradients are sums over all tokens: in the backward a workgroup keeps to query heads or
// to key heads, every lane adds its dims over the heads that it visits, the workgroup adds its lanes
// in LDS and writes one partial row, and a second launch adds the partials in workgroup order (no
// atomics: the same result every time).

#include <algorithm>
#include <type_traits>

#include "elem.hpp"
#include "fastdiv.hpp"

namespace soupk {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormWaves = kNormThreads / kWave;
constexpr int64_t kTwoGroups = 4096;                // wavefront items from which two are taken as one
constexpr int kNormBlocks = SOUPK_QK_NORM_BLOCKS;   // most workgroups (partial rows) of a backward

struct NormDims {
  int64_t rows, slots;  // tokens; B * T
  int T, NH, NKV, D;
  float inv_d;          // 1 / D
  int groups;           // wavefront items per token: ceil((NH + 2 NKV) * G / 64)
  FastDiv per_tok;      // divides by groups
  FastDiv per_seq;      // divides by T
};

template <int G>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (G >= 2) v = v + dpp_f<kDppQuad1032>(v);
  if constexpr (G >= 4) v = v + dpp_f<kDppQuad2301>(v);
  if constexpr (G >= 8) v = v + dpp_f<kDppHalfMirror>(v);
  if constexpr (G >= 16) v = v + dpp_f<kDppMirror>(v);
  return v;
}

__device__ __forceinline__ void load8f(const float* p, float* v) {
  Elem<float>::unpack8(Elem<float>::load8<false>(p), v);
}

// (The forward reads its rows through the caches -- the projection wrote them just before, and the
// backward comes back to them -- and the backward past them: forward + backward of 8192 tokens of 48
// heads 93.1 us, 96.2 with both cached.)
template <typename T, bool NT>
__device__ __forceinline__ void load16(const char* base, int64_t at, int half, float* a, float* b) {
  const auto ra = Elem<T>::template load8<NT>(base + at * Elem<T>::kBytes);
  const auto rb = Elem<T>::template load8<NT>(base + (at + half) * Elem<T>::kBytes);
  Elem<T>::unpack8(ra, a);
  Elem<T>::unpack8(rb, b);
}

// x += lora: fp32 deltas or deltas of the rows' type.
template <typename T, bool NT>
__device__ __forceinline__ void add_lora(const char* lora, bool f32, int64_t at, int half,
                                         float* a, float* b) {
  float la[8], lb[8];
  if (f32) load16<float, NT>(lora, at, half, la, lb);
  else load16<T, NT>(lora, at, half, la, lb);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    a[j] = a[j] + la[j];
    b[j] = b[j] + lb[j];
  }
}

__device__ __forceinline__ float sum_squares(const float* a, const float* b) {
  float s = a[0] * a[0], t = b[0] * b[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) {
    s = __builtin_fmaf(a[j], a[j], s);
    t = __builtin_fmaf(b[j], b[j], t);
  }
  return s + t;
}

// 1 / sqrt(mean + eps) by the hardware's reciprocal root (1 ulp).
__device__ __forceinline__ float inv_rms(float sum, float inv_d, float eps) {
  return __builtin_amdgcn_rsqf(__builtin_fmaf(sum, inv_d, eps));
}

// A wavefront takes PER neighbouring groups of 64 / G heads of one token (per_tok: such items per token).
template <typename T, int G, int PER>
__global__ __launch_bounds__(kNormThreads) void qk_norm_rope_fwd_kernel(
    const char* __restrict__ qkv, const char* __restrict__ lora_q, const char* __restrict__ lora_v,
    bool lora_f32, const float* __restrict__ wq, const float* __restrict__ wk,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t,
    const int64_t* __restrict__ pos, char* __restrict__ out, float eps, NormDims dm, uint32_t item0,
    uint32_t items) {
  constexpr int kSlots = kWave / G;                       // heads of a group
  const uint32_t item = item0 + blockIdx.x * kNormWaves + (threadIdx.x >> 6);
  if (item >= items) return;
  const int lane = threadIdx.x & 63, c = lane % G;
  const int heads = dm.NH + 2 * dm.NKV, half = dm.D >> 1;
  const uint32_t tok = dm.per_tok.div(item);
  const int h0 = static_cast<int>(item - tok * dm.per_tok.d) * (PER * kSlots) + lane / G;
  const int64_t ps = pos[tok];
  const bool known = ps >= 0 && ps < dm.slots;
  const int64_t at0 = (static_cast<int64_t>(tok) * heads + h0) * dm.D + 8 * c;
  const int64_t step = static_cast<int64_t>(kSlots) * dm.D;
  float a[PER][8], b[PER][8];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int h = h0 + u * kSlots;
#pragma unroll
    for (int j = 0; j < 8; ++j) a[u][j] = b[u][j] = 0.f;
    if (known && h < heads && 16 * c < dm.D) {
      load16<T, false>(qkv, at0 + u * step, half, a[u], b[u]);
      const bool is_q = h < dm.NH, is_v = h >= dm.NH + dm.NKV;
      const char* lora = is_q ? lora_q : (is_v ? lora_v : nullptr);
      if (lora != nullptr) {
        const int64_t row = is_q ? static_cast<int64_t>(tok) * dm.NH + h
                                 : static_cast<int64_t>(tok) * dm.NKV + (h - dm.NH - dm.NKV);
        add_lora<T, false>(lora, lora_f32, row * dm.D + 8 * c, half, a[u], b[u]);
      }
    }
  }
  float c1[8], c2[8], s1[8], s2[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c1[j] = c2[j] = s1[j] = s2[j] = 0.f;
  if (known && 16 * c < dm.D) {
    const uint32_t pu = static_cast<uint32_t>(ps);
    const uint32_t t = pu - dm.per_seq.div(pu) * dm.per_seq.d;
    const int64_t row = static_cast<int64_t>(t) * dm.D + 8 * c;
    load8f(cos_t + row, c1);
    load8f(cos_t + row + half, c2);
    load8f(sin_t + row, s1);
    load8f(sin_t + row + half, s2);
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int h = h0 + u * kSlots;
    const float ss = group_sum<G>(sum_squares(a[u], b[u]));
    if (h < heads && 16 * c < dm.D) {
      if (known && h < dm.NH + dm.NKV) {
        const float r = inv_rms(ss, dm.inv_d, eps);
        const float* w = (h < dm.NH ? wq : wk) + 8 * c;
        float w1[8], w2[8];
        load8f(w, w1);
        load8f(w + half, w2);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y1 = a[u][j] * r * w1[j], y2 = b[u][j] * r * w2[j];
          a[u][j] = __builtin_fmaf(y1, c1[j], -(y2 * s1[j]));
          b[u][j] = __builtin_fmaf(y2, c2[j], y1 * s2[j]);
        }
      }
      Elem<T>::template store8<true>(out + (at0 + u * step) * Elem<T>::kBytes, a[u]);
      Elem<T>::template store8<true>(out + (at0 + u * step + half) * Elem<T>::kBytes, b[u]);
    }
  }
}

// Workgroups [0, q_blocks) take the query heads (tokens * NH of them in order, q_per each), the others
// the key heads and, with each, the value head of the same number, whose gradient passes through.  So
// a lane needs one weight's sums only, and the weight stays in registers.
struct NormSplit {
  int q_blocks;
  uint32_t q_per, kv_per;      // heads of a workgroup
  FastDiv by_q, by_kv;         // divide by NH, NKV
};

template <typename T, int G, bool DW>
__global__ __launch_bounds__(kNormThreads) void qk_norm_rope_bwd_kernel(
    const char* __restrict__ dout, const char* __restrict__ qkv, const char* __restrict__ lora_q,
    bool lora_f32, const float* __restrict__ wq, const float* __restrict__ wk,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t,
    const int64_t* __restrict__ pos, char* __restrict__ dqkv, float* __restrict__ partial,
    float eps, NormDims dm, NormSplit sp) {
  constexpr int kSlots = kNormThreads / G;               // heads at a time
  const int half = dm.D >> 1;
  const int c = threadIdx.x % G, slot = threadIdx.x / G;
  const bool is_q = static_cast<int>(blockIdx.x) < sp.q_blocks;
  const FastDiv by = is_q ? sp.by_q : sp.by_kv;
  const uint32_t per = is_q ? sp.q_per : sp.kv_per;
  const uint32_t start = (is_q ? blockIdx.x : blockIdx.x - sp.q_blocks) * per;
  const uint32_t total = static_cast<uint32_t>(dm.rows) * by.d;
  const uint32_t end = min(total, start + per);
  const int heads = dm.NH + 2 * dm.NKV;
  const bool dims = 16 * c < dm.D;
  float w1[8], w2[8], acc1[8], acc2[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w1[j] = w2[j] = acc1[j] = acc2[j] = 0.f;
  if (dims) {
    load8f((is_q ? wq : wk) + 8 * c, w1);
    load8f((is_q ? wq : wk) + 8 * c + half, w2);
  }
  for (uint32_t i0 = start; i0 < end; i0 += kSlots) {
    const uint32_t i = i0 + slot;
    const bool live = i < end && dims;
    const uint32_t tok = by.div(live ? i : i0);
    const int h = static_cast<int>((live ? i : i0) - tok * by.d);
    const int64_t ps = pos[tok];
    const bool known = ps >= 0 && ps < dm.slots;
    const uint32_t pu = known ? static_cast<uint32_t>(ps) : 0u;
    const uint32_t t = pu - dm.per_seq.div(pu) * dm.per_seq.d;
    const int64_t at =
        (static_cast<int64_t>(tok) * heads + (is_q ? h : dm.NH + h)) * dm.D + 8 * c;
    const int64_t at_v = at + static_cast<int64_t>(dm.NKV) * dm.D;
    float a[8], b[8], g1[8], g2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = b[j] = g1[j] = g2[j] = 0.f;
    typename Elem<T>::Raw8 v1{}, v2{};
    if (live && known) {
      load16<T, true>(dout, at, half, g1, g2);
      load16<T, true>(qkv, at, half, a, b);
      if (!is_q) {
        v1 = Elem<T>::template load8<true>(dout + at_v * Elem<T>::kBytes);
        v2 = Elem<T>::template load8<true>(dout + (at_v + half) * Elem<T>::kBytes);
      }
      if (is_q && lora_q != nullptr)
        add_lora<T, true>(lora_q, lora_f32,
                          (static_cast<int64_t>(tok) * dm.NH + h) * dm.D + 8 * c, half, a, b);
    }
    const float r = inv_rms(group_sum<G>(sum_squares(a, b)), dm.inv_d, eps);
    float dot = 0.f;
    if (live && known) {
      const int64_t row = static_cast<int64_t>(t) * dm.D + 8 * c;
      float c1[8], c2[8], s1[8], s2[8];
      load8f(cos_t + row, c1);
      load8f(cos_t + row + half, c2);
      load8f(sin_t + row, s1);
      load8f(sin_t + row + half, s2);
      float d1 = 0.f, d2 = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y1 = __builtin_fmaf(g1[j], c1[j], g2[j] * s2[j]);
        const float y2 = __builtin_fmaf(g2[j], c2[j], -(g1[j] * s1[j]));
        a[j] = a[j] * r;
        b[j] = b[j] * r;
        if constexpr (DW) {
          acc1[j] = __builtin_fmaf(y1, a[j], acc1[j]);
          acc2[j] = __builtin_fmaf(y2, b[j], acc2[j]);
        }
        g1[j] = y1 * w1[j];
        g2[j] = y2 * w2[j];
        d1 = __builtin_fmaf(g1[j], a[j], d1);
        d2 = __builtin_fmaf(g2[j], b[j], d2);
      }
      dot = d1 + d2;
    }
    dot = group_sum<G>(dot) * dm.inv_d;
    if (live) {
      if (known) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g1[j] = r * __builtin_fmaf(-a[j], dot, g1[j]);
          g2[j] = r * __builtin_fmaf(-b[j], dot, g2[j]);
        }
      }
      Elem<T>::template store8<true>(dqkv + at * Elem<T>::kBytes, g1);
      Elem<T>::template store8<true>(dqkv + (at + half) * Elem<T>::kBytes, g2);
      if (!is_q) {
        st16<true>(dqkv + at_v * Elem<T>::kBytes, v1.w);
        st16<true>(dqkv + (at_v + half) * Elem<T>::kBytes, v2.w);
      }
    }
  }
  if constexpr (DW) {
    // The slots' sums of a dim are added in slot order.
    __shared__ float sum[kNormThreads * 8];
    float* const row = partial + static_cast<int64_t>(blockIdx.x) * dm.D;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j)
        sum[slot * (G * 8) + c * 8 + j] = part == 0 ? acc1[j] : acc2[j];
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < half) {          // (half <= G * 8)
        float s = 0.f;
#pragma unroll 8
        for (int k = 0; k < kSlots; ++k) s = s + sum[k * (G * 8) + threadIdx.x];
        row[part * half + threadIdx.x] = s;
      }
    }
  }
}

// dw = sum of the workgroups' rows in their order: per column 64 threads, each a stretch of the
// rows, joined in stretch order.  Columns [0, D) are the query weight's, [D, 2D) the key weight's.
constexpr int kSumCols = 4, kSumParts = kNormThreads / kSumCols;
__global__ __launch_bounds__(kNormThreads) void qk_norm_dw_kernel(
    const float* __restrict__ partial, int q_blocks, int blocks, int D, float* __restrict__ dwq,
    float* __restrict__ dwk) {
  __shared__ float s[kSumParts][kSumCols];
  const int col = threadIdx.x % kSumCols, part = threadIdx.x / kSumCols;
  const int x = blockIdx.x * kSumCols + col;               // (D is a multiple of 16)
  const bool is_q = x < D;
  const int b0 = is_q ? 0 : q_blocks, n = is_q ? q_blocks : blocks - q_blocks;
  const int per = (n + kSumParts - 1) / kSumParts;
  const float* const from = partial + static_cast<int64_t>(b0) * D + (is_q ? x : x - D);
  float v = 0.f;
  const int last = min(n, (part + 1) * per);
#pragma unroll 8
  for (int b = part * per; b < last; ++b) v = v + from[static_cast<int64_t>(b) * D];
  s[part][col] = v;
  __syncthreads();
  if (part != 0) return;
#pragma unroll 16
  for (int k = 1; k < kSumParts; ++k) v = v + s[k][col];
  float* const to = is_q ? dwq : dwk;
  if (to != nullptr) to[is_q ? x : x - D] = v;
}

// Calls f(integral constant G) with the lanes of a head of D dims.
template <typename F>
int with_group(int D, F&& f) {
  const int lanes = D / 16;
  if (lanes <= 1) return f(std::integral_constant<int, 1>{});
  if (lanes <= 2) return f(std::integral_constant<int, 2>{});
  if (lanes <= 4) return f(std::integral_constant<int, 4>{});
  if (lanes <= 8) return f(std::integral_constant<int, 8>{});
  return f(std::integral_constant<int, 16>{});
}

int group_of(int D) {
  int g = 1;
  while (g * 16 < D) g *= 2;
  return g;
}

// The shapes both directions take, or a status; fills dm and the wavefront items.
int norm_dims(int64_t rows, int32_t B, int32_t T, int32_t NH, int32_t NKV, int32_t D, float eps,
              NormDims& dm, int64_t& items) {
  if (rows < 0 || B < 0 || T < 0 || NH <= 0 || NKV < 0 || D <= 0 || D % 16 || D > 256)
    return kInvalid;
  if (!(eps >= 0.f) || eps > 3e38f) return kInvalid;
  if (static_cast<int64_t>(B) * T >= (int64_t{1} << 31) || NH > (1 << 16) || NKV > (1 << 16))
    return kInvalid;
  const int64_t heads = NH + 2 * static_cast<int64_t>(NKV);
  const int groups = static_cast<int>((heads * group_of(D) + kWave - 1) / kWave);
  // (32-bit indices of heads, with room for a last round)
  if (rows > ((int64_t{1} << 31) - 1 - (1 << 16)) / std::max<int64_t>(groups, heads)) return kInvalid;
  items = rows * groups;
  dm = NormDims{rows, static_cast<int64_t>(B) * T, T, NH, NKV, D, 1.0f / static_cast<float>(D), groups,
                FastDiv(static_cast<uint32_t>(groups)),
                FastDiv(static_cast<uint32_t>(std::max(T, 1)))};
  return kOk;
}

bool bad4(const void* p) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) & 3u); }

}  // namespace
}  // namespace soupk

using namespace soupk;

extern "C" __attribute__((visibility("default"))) int soupk_qk_norm_rope_fwd(
    const void* qkv, const void* lora_q, const void* lora_v, int32_t lora_dtype, const float* wq,
    const float* wk, const float* cos, const float* sin, const int64_t* pos, void* out,
    int32_t dtype, int64_t rows, int32_t B, int32_t T, int32_t NH, int32_t NKV, int32_t D,
    float eps, void* stream) {
  NormDims dm;
  int64_t items;
  if (norm_dims(rows, B, T, NH, NKV, D, eps, dm, items) != kOk) return kInvalid;
  if (dtype != SOUPK_DTYPE_F16 && dtype != SOUPK_DTYPE_BF16) return kInvalid;
  if ((lora_q || lora_v) && lora_dtype != dtype && lora_dtype != SOUPK_DTYPE_F32) return kInvalid;
  if (rows == 0) return kOk;
  if (bad_elem_ptr(qkv, dtype) || bad_elem_ptr(out, dtype) || bad4(wq) || bad4(wk)) return kInvalid;
  if (pos == nullptr || (reinterpret_cast<uintptr_t>(pos) & 7u)) return kInvalid;
  if (dm.slots > 0 && (bad4(cos) || bad4(sin))) return kInvalid;
  if ((lora_q && bad_elem_ptr(lora_q, lora_dtype)) || (lora_v && bad_elem_ptr(lora_v, lora_dtype)))
    return kInvalid;
  return with_type(dtype, [&](auto tag) -> int {
    using E = typename decltype(tag)::type;
    if constexpr (std::is_same_v<E, float>) {
      return kInvalid;
    } else {
      return with_group(D, [&](auto g) {
        constexpr int G = decltype(g)::value;
        auto run = [&](auto kernel, int per) {
          const int per_tok = (dm.groups + per - 1) / per;
          NormDims d = dm;
          d.per_tok = FastDiv(static_cast<uint32_t>(per_tok));
          const int64_t n = rows * per_tok;
          constexpr int64_t kMost = kMaxGrid * kNormWaves;      // of one launch
          for (int64_t i0 = 0; i0 < n; i0 += kMost) {
            const int64_t blocks = (std::min(kMost, n - i0) + kNormWaves - 1) / kNormWaves;
            const int rc = launch_kernel(
                kernel, dim3(static_cast<unsigned>(blocks)), dim3(kNormThreads),
                static_cast<hipStream_t>(stream), static_cast<const char*>(qkv),
                static_cast<const char*>(lora_q), static_cast<const char*>(lora_v),
                lora_dtype == SOUPK_DTYPE_F32, wq, wk, cos, sin, pos, static_cast<char*>(out), eps, d,
                static_cast<uint32_t>(i0), static_cast<uint32_t>(n));
            if (rc != kOk) return rc;
          }
          return static_cast<int>(kOk);
        };
        // Two groups a wavefront share the token's cos / sin loads, one a wavefront fills the chip
        // with fewer tokens: 8192 tokens of 48 heads 43.8 -> 40.1 us with two, 2048 of 16 heads
        // 5.9 -> 5.7, 888 of 16 heads 5.6 -> 6.5 (so not there).  (Fused multiply-adds and the
        // hardware's reciprocal root took the first from 40.1 to 38.5.)
        if (items >= kTwoGroups) return run(qk_norm_rope_fwd_kernel<E, G, 2>, 2);
        return run(qk_norm_rope_fwd_kernel<E, G, 1>, 1);
      });
    }
  });
}

extern "C" __attribute__((visibility("default"))) int soupk_qk_norm_rope_bwd(
    const void* dout, const void* qkv, const void* lora_q, int32_t lora_dtype, const float* wq,
    const float* wk, const float* cos, const float* sin, const int64_t* pos, void* dqkv,
    float* dwq, float* dwk, float* workspace, int64_t workspace_floats, int32_t dtype, int64_t rows,
    int32_t B, int32_t T, int32_t NH, int32_t NKV, int32_t D, float eps, void* stream) {
  NormDims dm;
  int64_t items;
  if (norm_dims(rows, B, T, NH, NKV, D, eps, dm, items) != kOk) return kInvalid;
  if (dtype != SOUPK_DTYPE_F16 && dtype != SOUPK_DTYPE_BF16) return kInvalid;
  if (lora_q && lora_dtype != dtype && lora_dtype != SOUPK_DTYPE_F32) return kInvalid;
  const bool want_dw = dwq != nullptr || dwk != nullptr;
  // Workgroups for the query heads and for the key and value heads, in proportion to what they
  // move; with weight gradients at most kNormBlocks in all (their partial rows).
  const int64_t slots = kNormThreads / group_of(D);
  const int64_t q_heads = rows * NH, kv_heads = rows * NKV;
  const int64_t q_need = (q_heads + slots - 1) / slots, kv_need = (kv_heads + slots - 1) / slots;
  const int64_t most = want_dw ? kNormBlocks : kMaxGrid / 2;    // (head numbers below 2^32)
  int64_t q_blocks = q_need, kv_blocks = kv_need;
  if (q_need + kv_need > most) {
    kv_blocks = std::min<int64_t>(kv_need, most * 5 * NKV / (3 * NH + 5 * NKV));
    if (NKV > 0) kv_blocks = std::max<int64_t>(kv_blocks, 1);
    q_blocks = std::min<int64_t>(q_need, most - kv_blocks);
  }
  auto share = [&](int64_t heads, int64_t blocks) {      // heads per workgroup, whole rounds
    return blocks > 0 ? ((heads + blocks - 1) / blocks + slots - 1) / slots * slots : slots;
  };
  const NormSplit sp{static_cast<int>(q_blocks), static_cast<uint32_t>(share(q_heads, q_blocks)),
                     static_cast<uint32_t>(share(kv_heads, kv_blocks)),
                     FastDiv(static_cast<uint32_t>(NH)),
                     FastDiv(static_cast<uint32_t>(std::max(NKV, 1)))};
  const int64_t blocks = q_blocks + kv_blocks;
  if (rows > 0) {
    if (bad_elem_ptr(dout, dtype) || bad_elem_ptr(qkv, dtype) || bad_elem_ptr(dqkv, dtype) ||
        bad4(wq) || bad4(wk))
      return kInvalid;
    if (pos == nullptr || (reinterpret_cast<uintptr_t>(pos) & 7u)) return kInvalid;
    if (dm.slots > 0 && (bad4(cos) || bad4(sin))) return kInvalid;
    if (lora_q && bad_elem_ptr(lora_q, lora_dtype)) return kInvalid;
  }
  if ((dwq && bad4(dwq)) || (dwk && bad4(dwk))) return kInvalid;
  if (want_dw && blocks > 0 && (bad4(workspace) || workspace_floats < blocks * D))
    return kInvalid;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows > 0) {
    const int rc = with_type(dtype, [&](auto tag) -> int {
      using E = typename decltype(tag)::type;
      if constexpr (std::is_same_v<E, float>) {
        return kInvalid;
      } else {
        return with_group(D, [&](auto g) {
          constexpr int G = decltype(g)::value;
          auto run = [&](auto kernel) {
            return launch_kernel(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kNormThreads), s,
                                 static_cast<const char*>(dout), static_cast<const char*>(qkv),
                                 static_cast<const char*>(lora_q), lora_dtype == SOUPK_DTYPE_F32,
                                 wq, wk, cos, sin, pos, static_cast<char*>(dqkv), workspace, eps,
                                 dm, sp);
          };
          return want_dw ? run(qk_norm_rope_bwd_kernel<E, G, true>)
                         : run(qk_norm_rope_bwd_kernel<E, G, false>);
        });
      }
    });
    if (rc != kOk) return rc;
  }
  if (!want_dw) return kOk;
  return launch_kernel(qk_norm_dw_kernel, dim3(2 * D / kSumCols), dim3(kNormThreads), s,
                       static_cast<const float*>(workspace), static_cast<int>(q_blocks),
                       static_cast<int>(blocks), static_cast<int>(D), dwq, dwk);
}
