// Verification of drafted tokens against the target's probabilities, from given random numbers
// (speculative sampling: Leviathan et al. 2023; Chen et al. 2023).
//
// Sequence b has L <= K drafted tokens x_i, drawn from the draft's rows q_i (or, without them, chosen
// with certainty: q_i is 1 at x_i), the target's rows p_0 .. p_K and numbers u_0 .. u_K in [0, 1):
//   x_i is accepted while u_i q_i(x_i) < p_i(x_i);   n: how many are, up to the first refusal
//   one more token is drawn from w = max(p_n - q_n, 0) after a refusal (from p_n where that is 0
//   everywhere), or from w = p_L when all were accepted: the lowest id whose prefix sum exceeds
//   u_K sum(w).
// The tokens kept have the target's distribution, whatever the draft's is.  The probabilities need not
// sum to one; a negative, infinite or NaN one counts as 0.
//
// Numbers: the products of the test are exact in fp64, and the sums are fp64: over 151936 columns fp32 sums
// would be off by more than the tokens' probabilities.  The order of the sums is fixed.
//
// Only the row that the token is drawn from is read (and the draft's): V elements a sequence.  Two
// launches: parts of a row are summed by a workgroup each, which finds n for itself (K reads); then one
// workgroup a sequence picks the part that holds the number and goes through that part alone.

#include <algorithm>
#include <type_traits>

#include "elem.hpp"

namespace soupk {
namespace {

constexpr int kThreads = 256;
constexpr int kRun = 16;                              // neighbouring elements of a thread when a part is searched
constexpr int kPart = kThreads * kRun;                // columns of a part, or a multiple
constexpr int kMostParts = kThreads;                  // of a row: one a thread of the second launch

struct VerifyArgs {
  const char* target;         // [B, K + 1, V]
  const char* draft;          // [B, K, V], or null
  const int64_t* tokens;      // [B, K]
  const float* uniforms;      // [B, K + 1]
  const int32_t* lengths;     // [B], or null
  double* sums;               // [B, parts, 2]: w, p
  int64_t* out;               // [B, K + 1]
  int32_t* accepted;          // [B]
  int64_t V, part;
  int B, K, parts;
};

__device__ __forceinline__ double mass(float v) { return v > 0.f && v < INFINITY ? static_cast<double>(v) : 0.0; }

// The number of tokens accepted, and whether a refusal ended them.  Every thread of a wavefront.
template <typename T>
__device__ __forceinline__ int accepted_of(const VerifyArgs& p, int b, bool& refused) {
  constexpr int E = Elem<T>::kBytes;
  const int lane = threadIdx.x & 63;
  const int len = p.lengths != nullptr ? min(max(p.lengths[b], 0), p.K) : p.K;
  for (int i0 = 0; i0 < len; i0 += kWave) {
    const int i = i0 + lane;
    bool stop = false;
    if (i < len) {
      const int64_t x = p.tokens[static_cast<int64_t>(b) * p.K + i];
      const bool known = x >= 0 && x < p.V;
      const int64_t at = known ? x : 0;
      const double px = mass(Elem<T>::load1(p.target + ((static_cast<int64_t>(b) * (p.K + 1) + i) * p.V + at) * E));
      double qx = 1.0;
      if (p.draft != nullptr)
        qx = mass(Elem<T>::load1(p.draft + ((static_cast<int64_t>(b) * p.K + i) * p.V + at) * E));
      const double u = p.uniforms[static_cast<int64_t>(b) * (p.K + 1) + i];
      stop = !(known && u * qx < px);
    }
    const uint64_t stops = __ballot(stop);
    if (stops != 0) {
      refused = true;
      return i0 + __ffsll(static_cast<unsigned long long>(stops)) - 1;
    }
  }
  refused = false;
  return len;
}

// What a column weighs: w, and p itself.
struct Row {
  const char* p;
  const char* q;              // null: nothing to take away
  int64_t one;                // the column whose weight is 0 (-1: none)
};
template <typename T>
__device__ __forceinline__ Row row_of(const VerifyArgs& a, int b, int n, bool refused) {
  constexpr int E = Elem<T>::kBytes;
  Row r{a.target + (static_cast<int64_t>(b) * (a.K + 1) + n) * a.V * E, nullptr, -1};
  if (refused) {
    if (a.draft != nullptr) r.q = a.draft + (static_cast<int64_t>(b) * a.K + n) * a.V * E;
    else r.one = a.tokens[static_cast<int64_t>(b) * a.K + n];
  }
  return r;
}
__device__ __forceinline__ double weight(float pv, float qv, bool one) {
  const double w = mass(pv) - mass(qv);
  return one || w < 0.0 ? 0.0 : w;
}

// Sum over the workgroup, in a fixed order; every thread gets it.
__device__ __forceinline__ double sum_threads(double v, double* scratch) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
  __syncthreads();
  return v;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a) {
  constexpr int E = Elem<T>::kBytes;
  __shared__ double scratch[kThreads / kWave];
  const int b = blockIdx.x / a.parts, part = blockIdx.x - b * a.parts;
  bool refused;
  const int n = accepted_of<T>(a, b, refused);
  const Row r = row_of<T>(a, b, n, refused);
  const int64_t c0 = part * a.part, c1 = min(c0 + a.part, a.V);
  double w = 0.0, p = 0.0;
  for (int64_t c = c0 + 8 * threadIdx.x; c < c1; c += 8 * kThreads) {
    float pv[8], qv[8];
    if (c + 8 <= c1) {
      Elem<T>::unpack8(Elem<T>::template load8<false>(r.p + c * E), pv);
      if (r.q != nullptr) Elem<T>::unpack8(Elem<T>::template load8<false>(r.q + c * E), qv);
    } else {
      for (int j = 0; j < 8; ++j) {
        pv[j] = c + j < c1 ? Elem<T>::load1(r.p + (c + j) * E) : 0.f;
        if (r.q != nullptr) qv[j] = c + j < c1 ? Elem<T>::load1(r.q + (c + j) * E) : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p += mass(pv[j]);
      w += weight(pv[j], r.q != nullptr ? qv[j] : 0.f, c + j == r.one);
    }
  }
  w = sum_threads(w, scratch);
  p = sum_threads(p, scratch);
  if (threadIdx.x == 0) {
    a.sums[2 * static_cast<int64_t>(blockIdx.x)] = w;
    a.sums[2 * static_cast<int64_t>(blockIdx.x) + 1] = p;
  }
}

// Inclusive prefix sum over the workgroup's threads; `before`: the sum of the threads before.
__device__ __forceinline__ double scan_threads(double v, double* scratch, double& before) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  double x = v;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const double o = __shfl_up(x, d);
    if (lane >= d) x += o;
  }
  double up = __shfl_up(x, 1);
  if (lane == 0) up = 0.0;
  if (lane == 63) scratch[w] = x;
  __syncthreads();
  double base = 0.0;
  for (int i = 0; i < w; ++i) base += scratch[i];
  __syncthreads();
  before = base + up;
  return base + x;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a) {
  constexpr int E = Elem<T>::kBytes;
  __shared__ double scratch[kThreads / kWave];
  __shared__ double found_base;
  __shared__ int first_part, last_part;
  __shared__ unsigned long long first_col, last_col;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  if (tid == 0) {
    first_part = kMostParts;
    last_part = -1;
    first_col = ~0ull;
    last_col = 0ull;
  }
  bool refused;
  const int n = accepted_of<T>(a, b, refused);
  Row r = row_of<T>(a, b, n, refused);
  const double* s = a.sums + 2 * (static_cast<int64_t>(b) * a.parts + tid);
  const double w = tid < a.parts ? s[0] : 0.0, p = tid < a.parts ? s[1] : 0.0;
  const bool from_p = !(sum_threads(w, scratch) > 0.0);
  if (from_p) r.q = nullptr, r.one = -1;
  const double mine = from_p ? p : w;
  double before;
  const double upto = scan_threads(mine, scratch, before);
  const double total = sum_threads(mine, scratch);
  // (the last thread's prefix, by which the numbers below are compared, in place of the other order's sum)
  __shared__ double whole;
  if (tid == kThreads - 1) whole = upto;
  __syncthreads();
  const double t = static_cast<double>(a.uniforms[static_cast<int64_t>(b) * (a.K + 1) + a.K]) * whole;
  int64_t drawn = -1;
  if (total > 0.0) {
    // the first part whose end passes t; rounding, or a number of 1 and more: the last one that weighs
    if (mine > 0.0) {
      if (upto > t) atomicMin(&first_part, tid);
      atomicMax(&last_part, tid);
    }
    __syncthreads();
    const int part = first_part < kMostParts ? first_part : last_part;
    if (tid == part) found_base = before;
    __syncthreads();
    double base = found_base;
    const int64_t c0 = part * a.part, c1 = min(c0 + a.part, a.V);
    for (int64_t at = c0; at < c1; at += kPart) {
      const int64_t c = at + kRun * tid;
      double sum = 0.0;
      double ws[kRun];
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        ws[j] = 0.0;
        if (c + j < c1)
          ws[j] = weight(Elem<T>::load1(r.p + (c + j) * E),
                         r.q != nullptr ? Elem<T>::load1(r.q + (c + j) * E) : 0.f, c + j == r.one);
        sum += ws[j];
      }
      double ahead;
      const double end = base + scan_threads(sum, scratch, ahead);
      double x = base + ahead;
      int first = kRun, last = -1;
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) last = last < 0 && ws[j] > 0.0 ? j : last;
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        x += ws[j];
        if (first == kRun && ws[j] > 0.0 && x > t) first = j;
      }
      // (one lane of a wavefront speaks for it: columns rise with the lanes)
      const uint64_t passed = __ballot(first < kRun), weighs = __ballot(last >= 0);
      if (passed != 0 && lane == __ffsll(static_cast<unsigned long long>(passed)) - 1)
        atomicMin(&first_col, static_cast<unsigned long long>(c + first));
      if (weighs != 0 && lane == 63 - __clzll(static_cast<long long>(weighs)))
        atomicMax(&last_col, static_cast<unsigned long long>(c + last));
      // (found, or on to the next columns of a long part: from the last thread's end)
      if (tid == kThreads - 1) found_base = end;
      __syncthreads();
      base = found_base;
      const bool done = first_col != ~0ull;
      __syncthreads();
      if (done) break;
    }
    drawn = static_cast<int64_t>(first_col != ~0ull ? first_col : last_col);
  }
  for (int i = tid; i <= a.K; i += kThreads) {
    int64_t v = -1;
    if (i < n) v = a.tokens[static_cast<int64_t>(b) * a.K + i];
    else if (i == n) v = drawn;
    a.out[static_cast<int64_t>(b) * (a.K + 1) + i] = v;
  }
  if (tid == 0) a.accepted[b] = n;
}

bool bad_ptr(const void* p, uintptr_t mask) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) & mask) != 0;
}

// Columns of a part (a multiple of kPart, kMostParts parts at most) and parts of a row.
void parts_of(int64_t V, int64_t& part, int& parts) {
  part = kPart;
  while ((V + part - 1) / part > kMostParts) part *= 2;
  parts = static_cast<int>((V + part - 1) / part);
}

}  // namespace
}  // namespace soupk

using namespace soupk;

extern "C" __attribute__((visibility("default"))) int soupk_verify_drafts_workspace(int64_t B, int64_t V,
                                                                                    int64_t* bytes) {
  if (bytes == nullptr || B < 0 || V < 1 || V >= (int64_t{1} << 40)) return kInvalid;
  int64_t part;
  int parts;
  parts_of(V, part, parts);
  if (B > kMaxGrid / parts) return kInvalid;
  *bytes = 16 * B * parts;
  return kOk;
}

extern "C" __attribute__((visibility("default"))) int soupk_verify_drafts(
    const void* target, const void* draft, int32_t dtype, const int64_t* tokens, const float* uniforms,
    const int32_t* lengths, int64_t* out, int32_t* accepted, int64_t B, int32_t K, int64_t V, void* workspace,
    int64_t workspace_bytes, void* stream) {
  int64_t need;
  if (K < 0 || K > (1 << 20) || soupk_verify_drafts_workspace(B, V, &need) != kOk) return kInvalid;
  if (B == 0) return kOk;
  if (bad_elem_ptr(target, dtype) || (draft != nullptr && bad_elem_ptr(draft, dtype)) || bad_ptr(uniforms, 3) ||
      bad_ptr(out, 7) || bad_ptr(accepted, 3) || bad_ptr(workspace, 7) || workspace_bytes < need ||
      (lengths != nullptr && bad_ptr(lengths, 3)) || (K > 0 && bad_ptr(tokens, 7)))
    return kInvalid;
  VerifyArgs a{static_cast<const char*>(target), static_cast<const char*>(draft), tokens, uniforms, lengths,
               static_cast<double*>(workspace), out, accepted, V, 0, static_cast<int>(B), K, 0};
  parts_of(V, a.part, a.parts);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto tag) -> int {
    using E = typename decltype(tag)::type;
    const int rc = launch_kernel(verify_sums_kernel<E>, dim3(static_cast<unsigned>(B * a.parts)), dim3(kThreads),
                                 s, a);
    if (rc != kOk) return rc;
    return launch_kernel(verify_pick_kernel<E>, dim3(static_cast<unsigned>(B)), dim3(kThreads), s, a);
  });
}
