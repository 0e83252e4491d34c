// Element types of kernels that take fp32, bf16 or f16 (MTC_DTYPE_*) and compute in fp32; runs of elements.
#pragma once

#include "mtc_attn.h"
#include "mtc_serve.h"

namespace mtc {
namespace attn {

template <int DT>
struct Value;
template <>
struct Value<MTC_DTYPE_F32> {
  typedef float type;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
template <>
struct Value<MTC_DTYPE_BF16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float get(uint16_t x) { return Elem<true>::widen(x); }
  static __device__ __forceinline__ uint16_t put(float x) { return Elem<true>::round(x); }
};
template <>
struct Value<MTC_DTYPE_F16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float get(uint16_t x) { return Elem<false>::widen(x); }
  static __device__ __forceinline__ uint16_t put(float x) { return Elem<false>::round(x); }
};

// N elements at an address that is a multiple of their size (up to 16 bytes), or of one element's only.
template <class T, int N>
struct __attribute__((aligned(sizeof(T) * N < 16 ? sizeof(T) * N : 16))) Run {
  T x[N];
};
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
  T x[N];
};

}  // namespace attn
}  // namespace mtc
