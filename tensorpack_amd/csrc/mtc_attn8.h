// Attention over the 8-bit cache, as mtc_cached_attention calls it (mtc_attn8.hip).
#pragma once

#include "mtc_cached.h"

namespace mtc {
namespace attn {

struct CodesCall : CachedCall {              // offsets in bytes
  const char* codes;
  int64_t page_bytes;
  int64_t k_codes, v_codes, k_scales, v_scales;      // of the layer's K and V within a page
  int32_t room;                              // bytes of a row
};
int run_codes(const CodesCall& a, bool bf, const CachedPlan& p, hipStream_t st);

}  // namespace attn
}  // namespace mtc
