// Device helpers of the attention kernels: element types, matrix instructions, global -> LDS copies,
// the LDS tile layouts, and one row computed by a plain loop.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mtc {
namespace attn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kOutOfRange = 0xFFFFFF00u;   // byte offset past any buffer's end
constexpr float kLog2e = 1.4426950408889634f;

// The two 16-bit types: BF true for bf16, false for f16.
//
// raise(lag): softmax weights that grow up to 2^lag over the running maximum are kept 2^raise larger than that, which drops out of
// the quotient. f16 has 5 exponent bits: a weight below 2^-14 loses bits and one below 2^-25 is zero. Raised to the top of the
// range (2^15), a row's weights lose less than 2^(lag - 40) of its largest one, each.
template <bool BF>
struct Elem;
template <>
struct Elem<true> {
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {      // round to nearest even
    x2 p = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, p);
  }
  static __device__ __forceinline__ float add2(uint32_t p, float s) {      // s + both elements of p, in fp32
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(x2, p), x2{(__bf16)1.0f, (__bf16)1.0f}, s, false);
  }
  static __device__ __forceinline__ uint16_t round(float a) { return __builtin_bit_cast(uint16_t, (__bf16)a); }
  static constexpr float raise(float) { return 0.0f; }
  static __device__ __forceinline__ float widen(uint16_t a) { return __builtin_bit_cast(float, (uint32_t)a << 16); }
};
template <>
struct Elem<false> {
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    x2 p = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, p);
  }
  static __device__ __forceinline__ float add2(uint32_t p, float s) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(x2, p), x2{(_Float16)1.0f, (_Float16)1.0f}, s, false);
  }
  static __device__ __forceinline__ uint16_t round(float a) { return __builtin_bit_cast(uint16_t, (_Float16)a); }
  static constexpr float raise(float lag) { return 15.0f - lag; }
  static __device__ __forceinline__ float widen(uint16_t a) { return (float)__builtin_bit_cast(_Float16, a); }
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// A raw buffer resource (uniform base, byte size).
__device__ __forceinline__ u32x4 buffer_rsrc(uint64_t base, uint32_t bytes) {
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)base),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(base >> 32) & 0xFFFFu)),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

// Global -> LDS copy of 16 bytes per lane: lane l's bytes land at lds + 16 l (lds uniform); a lane whose
// offset is past the buffer's end writes zeros, so the rows past a sequence's end hold zeros and
// nothing beyond it is read. Assembly, so the compiler does not make every LDS read wait for it: the
// kernels wait with counted s_waitcnt (the copies are their only vector memory loads in flight there). The wait states that
// the instruction needs are its own too, since the compiler adds none inside assembly: 1 after m0 is written, 5 after a
// vector instruction writes a scalar register that it reads (the resource by v_readfirstlane, or a spilled one by v_readlane).
__device__ __forceinline__ void copy16(u32x4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(voff), "s"(rsrc), "s"(lds)
               : "memory", "m0");
}

template <int N>
__device__ __forceinline__ void wait_copies() {       // at most N copies of this wave still in flight
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Workgroup barrier that orders LDS only (copies in flight stay in flight).
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Tiles in LDS: rows of DP elements (DP 64 or 128), cut into 16-byte pieces; piece c of row r lies at
// place c ^ key(r). The copies put it there by choosing each lane's source, so a row needs no padding.
// Two readings, one key each:
//   keys (K)    every lane one piece, the same c of consecutive rows: the rows must spread over the banks
//   values (V)  the transposing read: 32 lanes take 64 bytes of 4 consecutive rows (k_prompt) or 32 bytes of 8 (one wave's
//               keys): pairs of pieces stay together, 4 rows spread in steps of 64 bytes, 8 rows in steps of 32
template <int DP>
__device__ __forceinline__ uint32_t k_key(uint32_t row) {
  return DP == 128 ? (row & 15u) : ((row >> 1) & 7u);
}
template <int DP>
__device__ __forceinline__ uint32_t v_key(uint32_t row) {
  return DP == 128 ? (row & 3u) << 2 | (row & 4u) >> 1 : (row & 2u) << 1 | (row & 4u) >> 1;
}
__device__ __forceinline__ u32x4 lds_read16(uint32_t at) {
  return *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)at;
}
template <int DP>
__device__ __forceinline__ u32x4 read_k(const char* tile, uint32_t row, uint32_t piece) {
  return *reinterpret_cast<const u32x4*>(tile + row * (DP * 2) + ((piece ^ k_key<DP>(row)) << 4));
}

// Transposed read: of the 16 lanes that share `row4` (a multiple of 4) and `col16` (a multiple of 16), lane i gets
// elements (row4 .. row4+3, col16 + i). Lane i fetches 8 bytes: row row4 + i/4, columns col16 + 4 (i%4).
template <int DP>
__device__ __forceinline__ uint32_t v_place(uint32_t row4, uint32_t col16, uint32_t i) {
  const uint32_t row = row4 + (i >> 2), col = col16 + 4 * (i & 3);
  return row * (DP * 2) + (((col >> 3) ^ v_key<DP>(row)) << 4) + (col & 7) * 2;
}
__device__ __forceinline__ u32x2 lds_read_transposed(uint32_t at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)at));
}
template <int DP>
__device__ __forceinline__ u32x2 read_v(const char* tile, uint32_t row4, uint32_t col16, uint32_t i) {
  return lds_read_transposed(lds_addr(tile) + v_place<DP>(row4, col16, i));
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ bool finite(float x) { return (__builtin_bit_cast(uint32_t, x) & 0x7F800000u) != 0x7F800000u; }

template <class T>
__device__ __forceinline__ T wave_sum(T x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

// Maximum and sum over lanes l and l ^ 32: swapping the halves of two copies gives (low, low) and (high, high).
// (The results go through scalars: a bit cast of a vector's element takes the vector's first.)
__device__ __forceinline__ void both_halves(float x, float& low, float& high) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  low = __builtin_bit_cast(float, a);
  high = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float half_max(float x) {
  float low, high;
  both_halves(x, low, high);
  return fmaxf(low, high);
}
__device__ __forceinline__ float half_sum(float x) {
  float low, high;
  both_halves(x, low, high);
  return low + high;
}

template <bool BF>
__device__ __forceinline__ bool finite16(uint16_t x) {
  constexpr uint32_t exponent = BF ? 0x7F80u : 0x7C00u;
  return (x & exponent) != exponent;
}

// One row by a plain loop over its `seen` keys (one wave; lane l ends with o for dims l and l + 64). The tile
// kernels multiply keys that a row does not see by weights of 0, which is not 0 where V holds an infinity
// or a NaN: rows that come out not finite beside such keys are computed again here, where unseen keys are never read.
// From the last key back, so that a row that itself sees a NaN score (its result is NaN) mostly ends soon.
// kv(j) gives the addresses of key j's K and V (16-byte aligned rows).
template <bool BF, class KV>
__device__ void plain_row(const uint16_t* q, int dim, int seen, float c, KV kv, float& o0, float& o1) {
  const int lane = threadIdx.x & 63;
  auto score = [&](int j) {
    const uint16_t *k, *v;
    kv(j, k, v);
    float s = 0.0f;
    for (int d = 0; d < dim; d += 8) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(q + d), y = *reinterpret_cast<const u32x4*>(k + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = x[i], b = y[i];
        s = __builtin_fmaf(Elem<BF>::widen((uint16_t)a), Elem<BF>::widen((uint16_t)b), s);
        s = __builtin_fmaf(Elem<BF>::widen((uint16_t)(a >> 16)), Elem<BF>::widen((uint16_t)(b >> 16)), s);
      }
    }
    return s;
  };
  float top = -INFINITY;
  for (int j0 = seen; j0 > 0; j0 -= 64) {
    const int j = j0 - 1 - lane;
    const float s = j >= 0 ? score(j) : -INFINITY;
    if (__ballot(s != s)) {
      o0 = o1 = __builtin_nanf("");
      return;
    }
    top = fmaxf(top, s);
  }
  top = wave_max(top);
  float sum = 0.0f;
  o0 = o1 = 0.0f;
  for (int j0 = 0; j0 < seen; j0 += 64) {
    const float p = j0 + lane < seen ? exp2f((score(j0 + lane) - top) * c) : 0.0f;
    sum += p;
    const int n = min(64, seen - j0);
    for (int i = 0; i < n; ++i) {
      const uint16_t *k, *v;
      kv(j0 + i, k, v);
      const float w = __shfl(p, i);
      if (lane < dim) o0 = __builtin_fmaf(w, Elem<BF>::widen(v[lane]), o0);
      if (lane + 64 < dim) o1 = __builtin_fmaf(w, Elem<BF>::widen(v[lane + 64]), o1);
    }
  }
  sum = wave_sum(sum);
  if (sum == 0.0f) return;                         // no keys, or none with a weight: 0
  o0 /= sum;
  o1 /= sum;
}

}  // namespace attn
}  // namespace mtc
