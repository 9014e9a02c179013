// smoe_elt.h — the element types of the unquantised operators: 16-byte pieces
// of bf16, fp16 or fp32 rows as fp32 values and back.
//
// A row of any length may start at any multiple of its element size: gfx950
// serves a 16-byte access at such an address (the compiler emits the plain
// dwordx4 form for an under-aligned vector type), so odd row lengths need no
// kernel of their own, only a tail of single elements.
#pragma once

#include "smoe_common.h"

namespace smoe {

struct bf16_t {
  uint16_t u;
};
typedef _Float16 f16_t;
typedef uint32_t v4u_t __attribute__((ext_vector_type(4)));

template <class T>
struct Elt;

template <>
struct Elt<bf16_t> {
  static constexpr int kVec = 8, kDtype = SMOE_BF16;
  static __device__ __forceinline__ float to_f32(bf16_t x) { return __uint_as_float((uint32_t)x.u << 16); }
  static __device__ __forceinline__ bf16_t from_f32(float f) { return bf16_t{(uint16_t)bf16_pack2(f, 0.0f)}; }
  static __device__ __forceinline__ void unpack(const v4u_t& v, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ v4u_t pack(const float* f) {
    v4u_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = bf16_pack2(f[2 * i], f[2 * i + 1]);
    return v;
  }
};

template <>
struct Elt<f16_t> {
  static constexpr int kVec = 8, kDtype = SMOE_F16;
  static __device__ __forceinline__ float to_f32(f16_t x) { return (float)x; }
  static __device__ __forceinline__ f16_t from_f32(float f) { return (f16_t)f; }
  typedef f16_t v8h __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ void unpack(const v4u_t& v, float* f) {
    const v8h h = __builtin_bit_cast(v8h, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
  }
  static __device__ __forceinline__ v4u_t pack(const float* f) {
    v8h h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (f16_t)f[i];  // round to nearest even
    return __builtin_bit_cast(v4u_t, h);
  }
};

template <>
struct Elt<float> {
  static constexpr int kVec = 4, kDtype = SMOE_F32;
  static __device__ __forceinline__ float to_f32(float x) { return x; }
  static __device__ __forceinline__ float from_f32(float f) { return f; }
  static __device__ __forceinline__ void unpack(const v4u_t& v, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
  }
  static __device__ __forceinline__ v4u_t pack(const float* f) {
    v4u_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[i]);
    return v;
  }
};

// 16 bytes at any multiple of the element size.
typedef v4u_t v4u_under_t __attribute__((aligned(2)));
template <class T, bool kNT = false>
__device__ __forceinline__ v4u_t load_piece(const T* p) {
  if constexpr (kNT) return __builtin_nontemporal_load((const v4u_under_t*)p);
  else return *(const v4u_under_t*)p;
}
template <class T, bool kNT = false>
__device__ __forceinline__ void store_piece(T* p, const v4u_t& v) {
  if constexpr (kNT) __builtin_nontemporal_store(v, (v4u_under_t*)p);
  else *(v4u_under_t*)p = v;
}

// The first n (0 < n <= kVec) of a piece's values; the others read as 0 and
// are not stored.  Memory past the n elements is not touched.
template <class T, bool kNT = false>
__device__ __forceinline__ void load_f32(const T* p, int n, float* f) {
  constexpr int V = Elt<T>::kVec;
  if (n >= V) {
    Elt<T>::unpack(load_piece<T, kNT>(p), f);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = i < n ? Elt<T>::to_f32(p[i]) : 0.0f;
  }
}
template <class T, bool kNT = false>
__device__ __forceinline__ void store_f32(T* p, int n, const float* f) {
  constexpr int V = Elt<T>::kVec;
  if (n >= V) {
    store_piece<T, kNT>(p, Elt<T>::pack(f));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = Elt<T>::from_f32(f[i]);
  }
}

// The same as a raw piece.
template <class T>
__device__ __forceinline__ v4u_t load_some(const T* p, int n) {
  constexpr int V = Elt<T>::kVec;
  if (n >= V) return load_piece<T>(p);
  struct { T v[V]; } b;
#pragma unroll
  for (int i = 0; i < V; ++i) b.v[i] = i < n ? p[i] : T{};
  return __builtin_bit_cast(v4u_t, b);
}

// A parameter vector in the operands' type T or in fp32.
template <class T>
__device__ __forceinline__ void load_param(const void* p, bool f32, size_t i, int n, float* f) {
  constexpr int V = Elt<T>::kVec;
  if (f32) {
    load_f32<float>((const float*)p + i, n < 4 ? n : 4, f);
    if constexpr (V == 8) {
      if (n > 4) load_f32<float>((const float*)p + i + 4, n - 4, f + 4);
      else f[4] = f[5] = f[6] = f[7] = 0.0f;
    }
  } else {
    load_f32<T>((const T*)p + i, n, f);
  }
}

inline int elt_size(int dtype) { return dtype == SMOE_F32 ? 4 : 2; }

}  // namespace smoe

// An operand at a multiple of its element size, or NULL where that is allowed.
#define SMOE_CHECK_ELT(p, dtype)                                                          \
  do {                                                                                    \
    if ((p) == nullptr) return SMOE_EINVAL_NULL;                                          \
    if (((uintptr_t)(p)) & (uintptr_t)(smoe::elt_size(dtype) - 1)) return SMOE_EINVAL_PTRALIGN; \
  } while (0)
#define SMOE_CHECK_OPT(p, dtype)                                                          \
  do {                                                                                    \
    if (((uintptr_t)(p)) & (uintptr_t)(smoe::elt_size(dtype) - 1)) return SMOE_EINVAL_PTRALIGN; \
  } while (0)
