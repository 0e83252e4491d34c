// The 8-bit cache (MTC_CACHE_CODES8): where codes and scales lie in a page, and what a scale may be.
#pragma once

#include <stdint.h>

#include "mtc_serve.h"

namespace mtc {
namespace codes {

constexpr int kBlock = MTC_CODES8_BLOCK;                  // tokens of a scale

__host__ __device__ inline bool is_codes(const mtc_cache_desc& c) { return c.dtype & MTC_CACHE_CODES8; }
__host__ __device__ inline int base_type(const mtc_cache_desc& c) { return c.dtype & ~MTC_CACHE_CODES8; }

// Bytes of a token's row of codes, of all rows of a page, of a page.
__host__ __device__ inline int row_bytes(int dim) { return (dim + 15) & ~15; }
__host__ __device__ inline int64_t code_bytes(const mtc_cache_desc& c) {
  return 2ll * c.n_layers * c.kv_heads * c.page_size * row_bytes(c.dim);
}
__host__ __device__ inline int64_t page_bytes(const mtc_cache_desc& c) {
  return (code_bytes(c) + 4ll * c.n_layers * c.kv_heads * (c.page_size / kBlock) + 15) & ~15ll;
}

// Exponents: code 2^e is a number of the cache's type for every code of 8 bits. f16: 2^-24 is its smallest number, and
// 127 2^9 = 65024 lies below its largest, 65504. bf16 could go on to 2^-126 and 2^120; so far products of code, scale and q stay
// in fp32's range.
template <bool BF>
struct Range {
  static constexpr int lo = BF ? -100 : -24, hi = BF ? 100 : 9;
};

__device__ __forceinline__ float power(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
// A scale as memory holds it (whatever that is): at most 2^hi, not negative, not NaN. Without the lower bound, which products do not need.
template <bool BF>
__device__ __forceinline__ float scale_of(uint16_t bits) {
  return fminf(fmaxf(__builtin_bit_cast(float, (uint32_t)bits << 16), 0.0f), power(Range<BF>::hi));
}
template <bool BF>
__device__ __forceinline__ int exponent_of(uint16_t bits) {
  return min(max((int)(bits >> 7 & 0xFF) - 127, Range<BF>::lo), Range<BF>::hi);
}
// The smallest e with top <= 127 2^e (top = 1.m 2^x: 127 = 1.984375 2^6), within the range.
template <bool BF>
__device__ __forceinline__ int exponent_for(float top) {
  const uint32_t u = __builtin_bit_cast(uint32_t, top);
  const int e = (int)(u >> 23) - 127 - ((u & 0x7FFFFFu) <= 0x7E0000u ? 6 : 5);
  return min(max(e, Range<BF>::lo), Range<BF>::hi);
}

}  // namespace codes
}  // namespace mtc
