// Element types of the kernels that take fp16, bf16 or fp32 tensors: 8 consecutive elements to and
// from fp32 registers, at any element alignment.
//
// gfx950 runs with unaligned vector memory access enabled, so a row that starts at an odd element
// is read and written with the same 16-byte instructions as an aligned one (the types below tell
// the compiler that it may not assume more than the element's own alignment).
#pragma once

#include <type_traits>

#include "soupk_common.hpp"

namespace soupk {

typedef __bf16 bf16;

typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

// 16 bytes at any even address.
template <bool NT>
__device__ __forceinline__ u32x4 ld16(const void* p) {
  const u32x4_a2* q = static_cast<const u32x4_a2*>(p);
  if constexpr (NT) return __builtin_nontemporal_load(q);
  else return *q;
}
template <bool NT>
__device__ __forceinline__ void st16(void* p, u32x4 v) {
  u32x4_a2* q = static_cast<u32x4_a2*>(p);
  if constexpr (NT) __builtin_nontemporal_store(v, q);
  else *q = v;
}

__device__ __forceinline__ float bf2f(uint32_t bits16) {
  return __builtin_bit_cast(float, bits16 << 16);
}

// Two fp32 -> one dword of two bf16 (round to nearest even), `a` at the lower address; a and b are
// made opaque as in pack_h2.
__device__ __forceinline__ uint32_t pack_b2(float a, float b) {
  asm("" : "+v"(a), "+v"(b));
  typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
  bf16x2 v = {static_cast<bf16>(a), static_cast<bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}

typedef u32x2 u32x2_a2 __attribute__((aligned(2)));

// 8 bytes at any even address.
template <bool NT>
__device__ __forceinline__ u32x2 ld8(const void* p) {
  const u32x2_a2* q = static_cast<const u32x2_a2*>(p);
  if constexpr (NT) return __builtin_nontemporal_load(q);
  else return *q;
}
template <bool NT>
__device__ __forceinline__ void st8(void* p, u32x2 v) {
  u32x2_a2* q = static_cast<u32x2_a2*>(p);
  if constexpr (NT) __builtin_nontemporal_store(v, q);
  else *q = v;
}

// Elem<T>: T is the element as stored (f16, bf16, float).  kBytes of one element; Raw8, eight
// elements as loaded; load8 / unpack8 / store8 and the scalar forms.
template <typename T>
struct Elem;

template <typename T>
struct Elem16 {
  static constexpr int kBytes = 2;
  struct Raw8 {
    u32x4 w;
  };
  template <bool NT>
  static __device__ __forceinline__ Raw8 load8(const void* p) {
    return {ld16<NT>(p)};
  }
};

template <>
struct Elem<f16> : Elem16<f16> {
  static __device__ __forceinline__ void unpack8(const Raw8& r, float* v) {
    const u32x4 w = r.w;
    v[0] = lo_h(w.x); v[1] = hi_h(w.x); v[2] = lo_h(w.y); v[3] = hi_h(w.y);
    v[4] = lo_h(w.z); v[5] = hi_h(w.z); v[6] = lo_h(w.w); v[7] = hi_h(w.w);
  }
  template <bool NT>
  static __device__ __forceinline__ void store8(void* p, const float* v) {
    const u32x4 w = {pack_h2(v[0], v[1]), pack_h2(v[2], v[3]), pack_h2(v[4], v[5]),
                     pack_h2(v[6], v[7])};
    st16<NT>(p, w);
  }
  static __device__ __forceinline__ float load1(const void* p) {
    return h2f(*static_cast<const uint16_t*>(p));
  }
  static __device__ __forceinline__ void store1(void* p, float v) {
    *static_cast<uint16_t*>(p) = static_cast<uint16_t>(pack_h2(v, 0.f));
  }
};

template <>
struct Elem<bf16> : Elem16<bf16> {
  static __device__ __forceinline__ void unpack8(const Raw8& r, float* v) {
    const u32x4 w = r.w;
    v[0] = bf2f(w.x & 0xffffu); v[1] = bf2f(w.x >> 16);
    v[2] = bf2f(w.y & 0xffffu); v[3] = bf2f(w.y >> 16);
    v[4] = bf2f(w.z & 0xffffu); v[5] = bf2f(w.z >> 16);
    v[6] = bf2f(w.w & 0xffffu); v[7] = bf2f(w.w >> 16);
  }
  template <bool NT>
  static __device__ __forceinline__ void store8(void* p, const float* v) {
    const u32x4 w = {pack_b2(v[0], v[1]), pack_b2(v[2], v[3]), pack_b2(v[4], v[5]),
                     pack_b2(v[6], v[7])};
    st16<NT>(p, w);
  }
  static __device__ __forceinline__ float load1(const void* p) {
    return bf2f(*static_cast<const uint16_t*>(p));
  }
  static __device__ __forceinline__ void store1(void* p, float v) {
    *static_cast<uint16_t*>(p) = static_cast<uint16_t>(pack_b2(v, 0.f));
  }
};

template <>
struct Elem<float> {
  static constexpr int kBytes = 4;
  struct Raw8 {
    f32x4 a, b;
  };
  template <bool NT>
  static __device__ __forceinline__ Raw8 load8(const void* p) {
    const char* q = static_cast<const char*>(p);
    return {__builtin_bit_cast(f32x4, ld16<NT>(q)), __builtin_bit_cast(f32x4, ld16<NT>(q + 16))};
  }
  static __device__ __forceinline__ void unpack8(const Raw8& r, float* v) {
    v[0] = r.a.x; v[1] = r.a.y; v[2] = r.a.z; v[3] = r.a.w;
    v[4] = r.b.x; v[5] = r.b.y; v[6] = r.b.z; v[7] = r.b.w;
  }
  template <bool NT>
  static __device__ __forceinline__ void store8(void* p, const float* v) {
    char* q = static_cast<char*>(p);
    st16<NT>(q, __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}));
    st16<NT>(q + 16, __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]}));
  }
  static __device__ __forceinline__ float load1(const void* p) {
    return *static_cast<const float*>(p);
  }
  static __device__ __forceinline__ void store1(void* p, float v) { *static_cast<float*>(p) = v; }
};

// N = 4 or 8 consecutive elements to and from fp32.
template <typename T, int N, bool NT>
__device__ __forceinline__ void load_n(const char* p, float* v) {
  static_assert(N == 4 || N == 8, "");
  if constexpr (N == 8) {
    Elem<T>::unpack8(Elem<T>::template load8<NT>(p), v);
  } else if constexpr (std::is_same_v<T, float>) {
    const f32x4 f = __builtin_bit_cast(f32x4, ld16<NT>(p));
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
    const u32x2 w = ld8<NT>(p);
    if constexpr (std::is_same_v<T, f16>) {
      v[0] = lo_h(w.x); v[1] = hi_h(w.x); v[2] = lo_h(w.y); v[3] = hi_h(w.y);
    } else {
      v[0] = bf2f(w.x & 0xffffu); v[1] = bf2f(w.x >> 16);
      v[2] = bf2f(w.y & 0xffffu); v[3] = bf2f(w.y >> 16);
    }
  }
}
template <typename T, int N, bool NT>
__device__ __forceinline__ void store_n(char* p, const float* v) {
  static_assert(N == 4 || N == 8, "");
  if constexpr (N == 8)
    Elem<T>::template store8<NT>(p, v);
  else if constexpr (std::is_same_v<T, float>)
    st16<NT>(p, __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}));
  else if constexpr (std::is_same_v<T, f16>)
    st8<NT>(p, u32x2{pack_h2(v[0], v[1]), pack_h2(v[2], v[3])});
  else
    st8<NT>(p, u32x2{pack_b2(v[0], v[1]), pack_b2(v[2], v[3])});
}

// Most workgroups of a launch: HIP takes at most 2^32 - 1 threads along a grid's axis, and these kernels have
// up to 256 a workgroup (this leaves half of that for a launch of two kinds of them).
constexpr int64_t kMaxGrid = int64_t{1} << 23;

// Host: calls f(Elem type tag) for a SOUPK_DTYPE_* code; kInvalid for any other code.
template <typename T>
struct TypeTag {
  using type = T;
};
template <typename F>
int with_type(int32_t dtype, F&& f) {
  switch (dtype) {
    case SOUPK_DTYPE_F16: return f(TypeTag<f16>{});
    case SOUPK_DTYPE_BF16: return f(TypeTag<bf16>{});
    case SOUPK_DTYPE_F32: return f(TypeTag<float>{});
    default: return kInvalid;
  }
}

// True for a pointer that is null or not aligned to an element of the type.
inline bool bad_elem_ptr(const void* p, int32_t dtype) {
  const uintptr_t mask = dtype == SOUPK_DTYPE_F32 ? 3u : 1u;
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) & mask) != 0;
}

}  // namespace soupk
