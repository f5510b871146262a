// Element types of the row and rotary kernels: loads of VEC elements as fp32
// and stores rounded to nearest even (float32, bfloat16, float16).
#pragma once
#include "common.h"
#include "mfma.h"

template <int BYTES>
struct Words;
template <>
struct Words<16> { typedef uint4 type; };
template <>
struct Words<8> { typedef uint2 type; };
template <>
struct Words<4> { typedef uint32_t type; };
template <>
struct Words<2> { typedef uint16_t type; };

struct ElemF32 {
  typedef float type;
  static __device__ __forceinline__ float to_float(float v) { return v; }
  static __device__ __forceinline__ float from_float(float v) { return v; }
};
struct ElemBf16 {
  typedef __bf16 type;
  static __device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 from_float(float v) { return (__bf16)v; }
};
struct ElemF16 {
  typedef _Float16 type;
  static __device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 from_float(float v) { return (_Float16)v; }
};

// VEC elements of E as one memory access (E::type for VEC = 1)
template <class E, int VEC>
struct Pack {
  typedef typename E::type T;
  typedef typename Words<VEC * (int)sizeof(T)>::type W;
  union {
    W w;
    T e[VEC];
  };
  __device__ __forceinline__ Pack() {}
  static __device__ __forceinline__ Pack load(const void* p, int64_t i) {
    Pack r;
    r.w = *reinterpret_cast<const W*>(reinterpret_cast<const T*>(p) + i);
    return r;
  }
  __device__ __forceinline__ void store(void* p, int64_t i) const {
    *reinterpret_cast<W*>(reinterpret_cast<T*>(p) + i) = w;
  }
  __device__ __forceinline__ float get(int k) const { return E::to_float(e[k]); }
  __device__ __forceinline__ void set(int k, float v) { e[k] = E::from_float(v); }
};

inline int elem_size(int dtype) { return dtype == PRISM_F32 ? 4 : 2; }
