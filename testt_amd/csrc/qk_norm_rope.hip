// RMS norm of every query and key head with the position rotation in the same pass, into the
// token-major q|k|v rows that the varlen attention reads, and its backward.
//
// Per token and query or key head of D dims (the two halves of a head rotate against each other):
//   x = qkv (+ lora_q for a query head), r = 1 / sqrt(mean(x^2) + eps), n = x * r, y = n * w
//   out1 = y1 c1 - y2 s1, out2 = y2 c2 + y1 s2;   a value head passes through (+ lora_v)
// Backward, with g the gradient of out:
//   gy1 = g1 c1 + g2 s2, gy2 = g2 c2 - g1 s1;  dw = sum over tokens and heads of gy * n
//   dx = r * (gy w - n * mean(gy w n));        a value head's gradient passes through
// All in fp32, one rounding to the rows' type at the store; x and r are formed again in the
// backward from the rows it has to read anyway, so nothing is kept of the forward.
//
// Mapping: a head is a group of G = 2^k lanes, each with 8 dims of the first half and the 8 dims of
// the second half they rotate with, so the rotation is inside a lane and the mean of squares one
// DPP reduction of at most 16 lanes.  A wavefront takes 64 / G neighbouring heads of one token (8
// at D = 128): its loads and stores are whole rows of 2 KiB.  The token's cos / sin and the weight
// come from the caches.
//
// The weights' gradients are sums over all tokens: every lane adds its dims over the heads that it
// visits, a workgroup adds its lanes in LDS and writes one partial row, and a second launch adds the
// partials in workgroup order (no atomics: the same result every time).

#include <algorithm>
#include <type_traits>

#include "elem.hpp"
#include "fastdiv.hpp"

namespace soupk {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormWaves = kNormThreads / kWave;
constexpr int kNormBlocks = SOUPK_QK_NORM_BLOCKS;   // most workgroups (partial rows) of a backward

struct NormDims {
  int64_t rows, slots;  // tokens; B * T
  int T, NH, NKV, D;
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

// What a lane works on: 8 + 8 dims of one head of one token.
struct Place {
  bool live;        // a head and dims exist for this lane
  bool known;       // the token's position lies in [0, B*T)
  bool is_q, is_v;
  int64_t at;       // element of the first half in the q|k|v rows
  int64_t at_lora;  // the same in lora_q or lora_v
  const float *cos, *sin;
};

template <int G>
__device__ __forceinline__ Place place(uint32_t item, const NormDims& dm, const float* cos_t,
                                       const float* sin_t, const int64_t* pos) {
  const int lane = threadIdx.x & 63;
  const int c = lane % G;
  Place p;
  const uint32_t tok = dm.per_tok.div(item);
  const int h = static_cast<int>(item - tok * dm.per_tok.d) * (kWave / G) + lane / G;
  const int heads = dm.NH + 2 * dm.NKV;
  p.live = h < heads && 16 * c < dm.D;
  p.is_q = h < dm.NH;
  p.is_v = h >= dm.NH + dm.NKV;
  const int64_t ps = pos[tok];
  p.known = ps >= 0 && ps < dm.slots;
  const uint32_t pu = p.known ? static_cast<uint32_t>(ps) : 0u;
  const uint32_t t = pu - dm.per_seq.div(pu) * dm.per_seq.d;
  p.at = (static_cast<int64_t>(tok) * heads + h) * dm.D + 8 * c;
  p.at_lora = p.is_q ? (static_cast<int64_t>(tok) * dm.NH + h) * dm.D + 8 * c
                     : (static_cast<int64_t>(tok) * dm.NKV + (h - dm.NH - dm.NKV)) * dm.D + 8 * c;
  const int64_t row = static_cast<int64_t>(t) * dm.D + 8 * c;
  p.cos = cos_t + row;
  p.sin = sin_t + row;
  return p;
}

__device__ __forceinline__ void load8f(const float* p, float* v) {
  const f32x4_a4* q = reinterpret_cast<const f32x4_a4*>(p);
  const f32x4 a = q[0], b = q[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

template <typename T>
__device__ __forceinline__ void load16(const char* base, int64_t at, int half, float* a, float* b) {
  const auto ra = Elem<T>::template load8<true>(base + at * Elem<T>::kBytes);
  const auto rb = Elem<T>::template load8<true>(base + (at + half) * Elem<T>::kBytes);
  Elem<T>::unpack8(ra, a);
  Elem<T>::unpack8(rb, b);
}

// x += lora: fp32 deltas or deltas of the rows' type.
template <typename T>
__device__ __forceinline__ void add_lora(const char* lora, bool f32, int64_t at, int half,
                                         float* a, float* b) {
  float la[8], lb[8];
  if (f32) load16<float>(lora, at, half, la, lb);
  else load16<T>(lora, at, half, la, lb);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    a[j] = a[j] + la[j];
    b[j] = b[j] + lb[j];
  }
}

__device__ __forceinline__ float sum_squares(const float* a, const float* b) {
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = a[j] * a[j] + b[j] * b[j];
  return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

template <typename T, int G>
__global__ __launch_bounds__(kNormThreads) void qk_norm_rope_fwd_kernel(
    const char* __restrict__ qkv, const char* __restrict__ lora_q, const char* __restrict__ lora_v,
    bool lora_f32, const float* __restrict__ wq, const float* __restrict__ wk,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t,
    const int64_t* __restrict__ pos, char* __restrict__ out, float eps, NormDims dm,
    uint32_t items) {
  const uint32_t item = blockIdx.x * kNormWaves + (threadIdx.x >> 6);
  if (item >= items) return;
  const Place p = place<G>(item, dm, cos_t, sin_t, pos);
  const int half = dm.D >> 1;
  float a[8], b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.f;
  if (p.live && p.known) {
    load16<T>(qkv, p.at, half, a, b);
    const char* lora = p.is_q ? lora_q : (p.is_v ? lora_v : nullptr);
    if (lora != nullptr) add_lora<T>(lora, lora_f32, p.at_lora, half, a, b);
  }
  const float ss = group_sum<G>(sum_squares(a, b));
  if (!p.live) return;
  if (p.known && !p.is_v) {
    const float r = 1.0f / sqrtf(ss / static_cast<float>(dm.D) + eps);
    const float* w = (p.is_q ? wq : wk) + 8 * ((threadIdx.x & 63) % G);
    float w1[8], w2[8], c1[8], c2[8], s1[8], s2[8];
    load8f(w, w1);
    load8f(w + half, w2);
    load8f(p.cos, c1);
    load8f(p.cos + half, c2);
    load8f(p.sin, s1);
    load8f(p.sin + half, s2);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y1 = a[j] * r * w1[j], y2 = b[j] * r * w2[j];
      a[j] = y1 * c1[j] - y2 * s1[j];
      b[j] = y2 * c2[j] + y1 * s2[j];
    }
  }
  Elem<T>::template store8<true>(out + p.at * Elem<T>::kBytes, a);
  Elem<T>::template store8<true>(out + (p.at + half) * Elem<T>::kBytes, b);
}

template <typename T, int G, bool DW>
__global__ __launch_bounds__(kNormThreads) void qk_norm_rope_bwd_kernel(
    const char* __restrict__ dout, const char* __restrict__ qkv, const char* __restrict__ lora_q,
    bool lora_f32, const float* __restrict__ wq, const float* __restrict__ wk,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t,
    const int64_t* __restrict__ pos, char* __restrict__ dqkv, float* __restrict__ partial,
    float eps, NormDims dm, uint32_t items) {
  const int half = dm.D >> 1;
  const int c = (threadIdx.x & 63) % G;
  float acc[32];     // [q: first half, second half | k: first half, second half]
  if constexpr (DW) {
#pragma unroll
    for (int j = 0; j < 32; ++j) acc[j] = 0.f;
  }
  const uint32_t stride = gridDim.x * kNormWaves;
  for (uint32_t item = blockIdx.x * kNormWaves + (threadIdx.x >> 6); item < items;
       item += stride) {
    const Place p = place<G>(item, dm, cos_t, sin_t, pos);
    float a[8], b[8], g1[8], g2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = b[j] = g1[j] = g2[j] = 0.f;
    const bool norm = p.live && p.known && !p.is_v;
    if (p.live && p.known) load16<T>(dout, p.at, half, g1, g2);
    if (norm) {
      load16<T>(qkv, p.at, half, a, b);
      if (p.is_q && lora_q != nullptr) add_lora<T>(lora_q, lora_f32, p.at_lora, half, a, b);
    }
    const float r =
        1.0f / sqrtf(group_sum<G>(sum_squares(a, b)) / static_cast<float>(dm.D) + eps);
    float dot = 0.f;
    if (norm) {
      const float* w = (p.is_q ? wq : wk) + 8 * c;
      float w1[8], w2[8], c1[8], c2[8], s1[8], s2[8];
      load8f(w, w1);
      load8f(w + half, w2);
      load8f(p.cos, c1);
      load8f(p.cos + half, c2);
      load8f(p.sin, s1);
      load8f(p.sin + half, s2);
      float d1 = 0.f, d2 = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y1 = g1[j] * c1[j] + g2[j] * s2[j];
        const float y2 = g2[j] * c2[j] - g1[j] * s1[j];
        a[j] = a[j] * r;
        b[j] = b[j] * r;
        const float t1 = y1 * a[j], t2 = y2 * b[j];
        if constexpr (DW) {
          acc[j] = acc[j] + (p.is_q ? t1 : 0.f);
          acc[8 + j] = acc[8 + j] + (p.is_q ? t2 : 0.f);
          acc[16 + j] = acc[16 + j] + (p.is_q ? 0.f : t1);
          acc[24 + j] = acc[24 + j] + (p.is_q ? 0.f : t2);
        }
        g1[j] = y1 * w1[j];
        g2[j] = y2 * w2[j];
        d1 = d1 + g1[j] * a[j];
        d2 = d2 + g2[j] * b[j];
      }
      dot = d1 + d2;
    }
    dot = group_sum<G>(dot) / static_cast<float>(dm.D);
    if (!p.live) continue;
    if (norm) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g1[j] = r * (g1[j] - a[j] * dot);
        g2[j] = r * (g2[j] - b[j] * dot);
      }
    }
    Elem<T>::template store8<true>(dqkv + p.at * Elem<T>::kBytes, g1);
    Elem<T>::template store8<true>(dqkv + (p.at + half) * Elem<T>::kBytes, g2);
  }
  if constexpr (DW) {
    // The lanes of one c hold the same dims: they are added in the order of the thread index.
    constexpr int kPer = kNormThreads / G;               // lanes per c
    __shared__ float sum[kNormThreads * 8 + 8];
    const int who = threadIdx.x / G;
    float* const row = partial + static_cast<int64_t>(blockIdx.x) * 2 * dm.D;
    for (int part = 0; part < 4; ++part) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = part == 0 ? acc[j] : part == 1 ? acc[8 + j] : part == 2 ? acc[16 + j]
                                                                            : acc[24 + j];
        sum[who * (G * 8) + c * 8 + j] = v;
      }
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < half) {          // (half <= G * 8)
        float s = 0.f;
        for (int k = 0; k < kPer; ++k) s = s + sum[k * (G * 8) + threadIdx.x];
        row[(part >> 1) * dm.D + (part & 1) * half + threadIdx.x] = s;
      }
    }
  }
}

// dw = sum of the partial rows in workgroup order: 16 threads per column, each a stretch of the
// rows, joined in stretch order.
constexpr int kSumCols = 16, kSumParts = 16;
__global__ __launch_bounds__(kSumCols* kSumParts) void qk_norm_dw_kernel(
    const float* __restrict__ partial, int blocks, int D, float* __restrict__ dwq,
    float* __restrict__ dwk) {
  __shared__ float s[kSumParts][kSumCols];
  const int col = threadIdx.x % kSumCols, part = threadIdx.x / kSumCols;
  const int x = blockIdx.x * kSumCols + col;
  const int per = (blocks + kSumParts - 1) / kSumParts;
  float v = 0.f;
  if (x < 2 * D)
    for (int b = part * per; b < min(blocks, (part + 1) * per); ++b)
      v = v + partial[static_cast<int64_t>(b) * 2 * D + x];
  s[part][col] = v;
  __syncthreads();
  if (part != 0 || x >= 2 * D) return;
  for (int k = 1; k < kSumParts; ++k) v = v + s[k][col];
  float* const to = x < D ? dwq : dwk;
  if (to != nullptr) to[x < D ? x : x - D] = v;
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
  if (rows > ((int64_t{1} << 31) - 1 - kNormWaves * kNormBlocks) / groups) return kInvalid;
  items = rows * groups;
  dm = NormDims{rows, static_cast<int64_t>(B) * T, T,  NH, NKV, D, groups,
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
        const dim3 grid(static_cast<unsigned>((items + kNormWaves - 1) / kNormWaves));
        return launch_kernel(qk_norm_rope_fwd_kernel<E, decltype(g)::value>, grid,
                             dim3(kNormThreads), static_cast<hipStream_t>(stream),
                             static_cast<const char*>(qkv), static_cast<const char*>(lora_q),
                             static_cast<const char*>(lora_v), lora_dtype == SOUPK_DTYPE_F32, wq,
                             wk, cos, sin, pos, static_cast<char*>(out), eps, dm,
                             static_cast<uint32_t>(items));
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
  const int64_t blocks =
      std::min<int64_t>(kNormBlocks, (items + kNormWaves - 1) / kNormWaves);
  if (rows > 0) {
    if (bad_elem_ptr(dout, dtype) || bad_elem_ptr(qkv, dtype) || bad_elem_ptr(dqkv, dtype) ||
        bad4(wq) || bad4(wk))
      return kInvalid;
    if (pos == nullptr || (reinterpret_cast<uintptr_t>(pos) & 7u)) return kInvalid;
    if (dm.slots > 0 && (bad4(cos) || bad4(sin))) return kInvalid;
    if (lora_q && bad_elem_ptr(lora_q, lora_dtype)) return kInvalid;
  }
  if ((dwq && bad4(dwq)) || (dwk && bad4(dwk))) return kInvalid;
  if (want_dw && blocks > 0 && (bad4(workspace) || workspace_floats < blocks * 2 * D))
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
          auto run = [&](auto kernel, int64_t n) {
            return launch_kernel(kernel, dim3(static_cast<unsigned>(n)), dim3(kNormThreads), s,
                                 static_cast<const char*>(dout), static_cast<const char*>(qkv),
                                 static_cast<const char*>(lora_q), lora_dtype == SOUPK_DTYPE_F32,
                                 wq, wk, cos, sin, pos, static_cast<char*>(dqkv), workspace, eps,
                                 dm, static_cast<uint32_t>(items));
          };
          return want_dw ? run(qk_norm_rope_bwd_kernel<E, G, true>, blocks)
                         : run(qk_norm_rope_bwd_kernel<E, G, false>,
                               (items + kNormWaves - 1) / kNormWaves);
        });
      }
    });
    if (rc != kOk) return rc;
  }
  if (!want_dw) return kOk;
  return launch_kernel(qk_norm_dw_kernel, dim3((2 * D + kSumCols - 1) / kSumCols),
                       dim3(kSumCols * kSumParts), s, static_cast<const float*>(workspace),
                       static_cast<int>(blocks), static_cast<int>(D), dwq, dwk);
}
