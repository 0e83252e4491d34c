"""Where cached attention's count of units leaves 32 bits (include/mtc_serve.h): host-side, without a GPU."""

import ctypes

import pytest

from tensorpack_amd import _abi, _native


@pytest.mark.parametrize("codes,start", [(0, 4), (_abi.CACHE_CODES8, 5)])
@pytest.mark.parametrize("heads,tokens,slots", [(2, 1, 2048 + 2 * 8192), (40, 2, 512 + 2 * 8192), (64, 1, 2048 + 2 * 8192)])
def test_largest_capacity(codes, start, heads, tokens, slots):
    """8192 sequences of two K/V heads: a unit of 32 keys, one for a part of a unit, and the start of an item (4 units, 5 over codes), times the
    partial results that there may be (a run of each of 512 blocks, or of their 4 waves, and an item of each sequence and head)."""
    lib = _native.hip_lib()
    page = 32
    units = 0x7FFFFFFF // slots
    for pages, accepted in ((units - 1 - start, True), (units - start, False)):
        c = _abi.MtcCacheDesc(_abi.ABI_VERSION, _abi.MTC_DTYPE_BF16 | codes, 100, 1, 2, 64, page, 8192, pages, 0, 0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000)
        h = _abi.MtcHeads(0x1000, heads * 64, 64)
        a = _abi.MtcCachedArgs(_abi.ABI_VERSION, 0, 8192, tokens, heads, 0, 0.125, 0, h, h, 0x7000, None, None, None)
        assert lib.mtc_check_cache_desc(ctypes.byref(c)) == 0
        need = lib.mtc_cached_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(a))
        assert (need > 0) == accepted, (pages, need)
        if not accepted:
            assert b"too much for one call" in lib.mtc_last_error()
