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
// launches: parts of a row are summed by a wavefront each, which finds n for itself (K reads); then one
// workgroup a sequence picks the part that holds the number and goes through its 1024 columns alone.
//
// MI355X, 64 sequences of 8 drafts and 151936 fp32 columns: 17.1 us, of which the sums (63 MB, half the rows
// refused) 14.1 and the pick 3.9.  One sequence: 4.4 and 3.0, latency (tokens, their probabilities, the row,
// one after another).  A wavefront's row in flight 512 columns at a time: eight wavefronts a SIMD; 1024 at a
// time 18.9 instead of 18.4 us then, and 16.5 instead of 15.0 for bf16; parts of 2048 columns 20.0 / 18.2.

#include <algorithm>
#include <type_traits>

#include "elem.hpp"

namespace soupk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kRun = 4;                               // neighbouring columns of a thread when a part is searched
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
  for (int i0 = 0; i0 < p.K; i0 += kWave) {
    // (read whether it counts or not: its length is on its way too)
    const int i = min(i0 + lane, p.K - 1);
    const int64_t x = p.tokens[static_cast<int64_t>(b) * p.K + i];
    const double u = p.uniforms[static_cast<int64_t>(b) * (p.K + 1) + i];
    const bool known = x >= 0 && x < p.V;
    const int64_t at = known ? x : 0;
    const double px = mass(Elem<T>::load1(p.target + ((static_cast<int64_t>(b) * (p.K + 1) + i) * p.V + at) * E));
    double qx = 1.0;
    if (p.draft != nullptr)
      qx = mass(Elem<T>::load1(p.draft + ((static_cast<int64_t>(b) * p.K + i) * p.V + at) * E));
    const uint64_t stops = __ballot(i0 + lane < len && !(known && u * qx < px));
    if (stops != 0) {
      refused = true;
      return i0 + __ffsll(static_cast<unsigned long long>(stops)) - 1;
    }
    if (i0 + kWave >= len) break;
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

// v of another lane, by DPP (0 in rows of 16 outside ROWS, and where there is no such lane).
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Inclusive prefix sum over the wavefront's lanes: within rows of 16 from 1, 2, 4 and 8 lanes before, then the last
// lane of a row for the next one and of the first half for the second.
__device__ __forceinline__ double scan_lanes(double v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}

// A wavefront a part.  (One of a workgroup's finding n for all: 16.6 to 19.5 us instead of 16.6 for 64 bf16
// rows, with 4 to 16 wavefronts.)
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a) {
  constexpr int E = Elem<T>::kBytes;
  const int groups = (a.parts + kWaves - 1) / kWaves;
  const int b = blockIdx.x / groups, lane = threadIdx.x & 63;
  const int part = (blockIdx.x - b * groups) * kWaves + (threadIdx.x >> 6);
  if (part >= a.parts) return;
  bool refused;
  const int n = accepted_of<T>(a, b, refused);
  const Row r = row_of<T>(a, b, n, refused);
  const int64_t c0 = part * a.part, c1 = min(c0 + a.part, a.V);
  double w = 0.0, p = 0.0;
#pragma unroll 1
  for (int64_t c = c0 + 8 * lane; c < c1; c += 8 * kWave) {
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
  w = scan_lanes(w);
  p = scan_lanes(p);
  if (lane == kWave - 1) {
    double* out = a.sums + 2 * (static_cast<int64_t>(b) * a.parts + part);
    out[0] = w;
    out[1] = p;
    if (part == 0) a.accepted[b] = n;
  }
}

// Inclusive prefix sum over the workgroup's threads; `before`: the sum of the threads before, `all`: of all.
__device__ __forceinline__ double scan_threads(double v, double* scratch, double& before, double& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const double x = scan_lanes(v), up = moved<0x138, 0xf>(x);
  __syncthreads();
  if (lane == 63) scratch[w] = x;
  __syncthreads();
  double base = 0.0;
  all = 0.0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i == w) base = all;
    all += scratch[i];
  }
  before = base + up;
  return base + x;
}

// The first thread whose `passed` is set (kThreads: none), and the last whose `weighs` is (-1: none).
__device__ __forceinline__ int first_of(bool passed, bool weighs, int* scratch, int& last) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t p = __ballot(passed), g = __ballot(weighs);
  __syncthreads();
  if (lane == 0) {
    scratch[w] = p != 0 ? kWave * w + __ffsll(static_cast<unsigned long long>(p)) - 1 : kThreads;
    scratch[kWaves + w] = g != 0 ? kWave * w + 63 - __clzll(static_cast<long long>(g)) : -1;
  }
  __syncthreads();
  int first = kThreads;
  last = -1;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    first = min(first, scratch[i]);
    last = max(last, scratch[kWaves + i]);
  }
  return first;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a) {
  constexpr int E = Elem<T>::kBytes;
  __shared__ double scratch[kWaves];
  __shared__ int marks[2 * kWaves];
  __shared__ double found_base;
  __shared__ long long found_col[2];        // the column, and the last one that weighs
  const int b = blockIdx.x, tid = threadIdx.x;
  const int n = a.accepted[b];
  const int len = a.lengths != nullptr ? min(max(a.lengths[b], 0), a.K) : a.K;
  const double* s = a.sums + 2 * (static_cast<int64_t>(b) * a.parts + min(tid, a.parts - 1));
  const double w = tid < a.parts ? s[0] : 0.0, p = tid < a.parts ? s[1] : 0.0;
  const double number = a.uniforms[static_cast<int64_t>(b) * (a.K + 1) + a.K];
  for (int i = tid; i <= a.K; i += kThreads)
    if (i != n)
      a.out[static_cast<int64_t>(b) * (a.K + 1) + i] =
          i < n ? a.tokens[static_cast<int64_t>(b) * a.K + i] : -1;
  Row r = row_of<T>(a, b, n, n < len);
  double before, total, mine = w;
  double upto = scan_threads(mine, scratch, before, total);
  if (!(total > 0.0)) {                     // nothing is left of the target's row: the row itself
    r.q = nullptr;
    r.one = -1;
    mine = p;
    upto = scan_threads(mine, scratch, before, total);
  }
  int64_t drawn = -1;
  if (total > 0.0) {
    const double t = number * total;
    // the first part whose end passes t; by rounding, or for a number of 1 and more: the last one that weighs
    int last;
    const int first = first_of(mine > 0.0 && upto > t, mine > 0.0, marks, last);
    const int part = first < kThreads ? first : last;
    if (tid == part) found_base = before;
    if (tid == 0) found_col[0] = found_col[1] = -1;
    __syncthreads();
    double base = found_base;
    const int64_t c0 = part * a.part, c1 = min(c0 + a.part, a.V);
    for (int64_t at = c0; at < c1; at += kPart) {
      const int64_t c = at + kRun * tid;
      float pv[kRun], qv[kRun];
      if (c + kRun <= c1) {
        load_n<T, kRun, false>(r.p + c * E, pv);
        if (r.q != nullptr) load_n<T, kRun, false>(r.q + c * E, qv);
      } else {
        for (int j = 0; j < kRun; ++j) {
          pv[j] = c + j < c1 ? Elem<T>::load1(r.p + (c + j) * E) : 0.f;
          if (r.q != nullptr) qv[j] = c + j < c1 ? Elem<T>::load1(r.q + (c + j) * E) : 0.f;
        }
      }
      double ws[kRun], sum = 0.0;
      int first_j = kRun, last_j = -1;
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        ws[j] = weight(pv[j], r.q != nullptr ? qv[j] : 0.f, c + j == r.one);
        sum += ws[j];
        if (ws[j] > 0.0) last_j = j;
      }
      double ahead, all;
      scan_threads(sum, scratch, ahead, all);
      double x = base + ahead;
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        x += ws[j];
        if (first_j == kRun && ws[j] > 0.0 && x > t) first_j = j;
      }
      int last_thread;
      const int thread = first_of(first_j < kRun, last_j >= 0, marks, last_thread);
      if (tid == thread) found_col[0] = c + first_j;
      if (tid == last_thread) found_col[1] = c + last_j;
      __syncthreads();
      if (thread < kThreads) break;
      base += all;                          // (on to the next columns of a long part)
    }
    drawn = found_col[0] >= 0 ? found_col[0] : found_col[1];
  }
  if (tid == 0) a.out[static_cast<int64_t>(b) * (a.K + 1) + n] = drawn;
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
    const int rc = launch_kernel(verify_sums_kernel<E>,
                                 dim3(static_cast<unsigned>(B * ((a.parts + kWaves - 1) / kWaves))), dim3(kThreads),
                                 s, a);
    if (rc != kOk) return rc;
    return launch_kernel(verify_pick_kernel<E>, dim3(static_cast<unsigned>(B)), dim3(kThreads), s, a);
  });
}
