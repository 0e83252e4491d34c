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

// Maximum over the wave, in every lane (row shifts, then the rows' maxima): an eighth of the time of exchanges through LDS.
template <class Max>
__device__ __forceinline__ uint32_t wave_most(uint32_t x, Max most) {
  x = most(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xF, 0xF, false));
  x = most(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xF, 0xF, false));
  x = most(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xF, 0xF, false));
  x = most(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xF, 0xF, false));
  x = most(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xA, 0xF, false));      // row_bcast:15 into rows 1 and 3
  x = most(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xC, 0xF, false));      // row_bcast:31 into rows 2 and 3
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ float wave_top(float x) {
  auto most = [](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
  };
  return __builtin_bit_cast(float, wave_most(__builtin_bit_cast(uint32_t, x), most));
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
  return wave_most(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

}  // namespace attn
}  // namespace mtc
