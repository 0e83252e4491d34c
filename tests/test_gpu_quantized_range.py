"""cached_attention over a QuantizedCache at the ends of what its scales, its queries and its table may hold, against the definition in
64 bits with the bar of test_gpu_attention. Each in all three ways through the keys: up to 16 rows, up to 32, and more."""

import math

import numpy as np
import pytest

from test_gpu_attention import _check, _dtype, _ints, _normal, _rows64
from test_gpu_quantized_attention import _cache

pytestmark = pytest.mark.gpu
WAYS = [(1, 8), (4, 8), (12, 8)]                                   # tokens, heads of one K/V head


@pytest.mark.parametrize("tokens,heads", WAYS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_pages_that_do_not_exist(gpu, dtype, tokens, heads):
    """Tokens on no page count as zeros, whatever the scales in memory are."""
    from tensorpack_amd.attention import cached_attention
    lens, page = [100, 70], 16
    cache = _cache(gpu, lens, page, 1, 64, dtype, layers=1, junk=False)
    spare = next(p for p in range(1, cache.n_pages) if not (cache.table == p).any())
    cache.copy_pages(_ints([0], gpu), _ints([spare], gpu))
    cache.table[cache.table == 0] = spare                           # page 0 is nobody's
    codes, scales = cache.codes[:, 0].cpu().numpy().astype(np.float64), cache.scales[:, 0].double().cpu().numpy()
    cache.table[0, 2], cache.table[0, 4], cache.table[1, 0] = -1, 1 << 30, cache.n_pages
    table = cache.table.cpu().numpy()
    q = _normal(9, (2, tokens, heads, 64), _dtype(dtype), gpu, 2.0)
    qq = q.double().cpu().numpy()
    o, A = np.zeros(qq.shape), np.zeros(qq.shape)
    for b, n in enumerate(lens):
        at = np.arange(n)
        p = table[b][at // page]
        good = (p >= 0) & (p < cache.n_pages)
        p = np.where(good, p, 0)
        k, v = (np.where(good[:, None], codes[p, j, 0, at % page] * scales[p, j, 0, 0][:, None], 0.0) for j in (0, 1))
        for h in range(heads):
            o[b, :, h], A[b, :, h] = _rows64(qq[b, :, h], k, v, [n - tokens + t + 1 for t in range(tokens)], 0.125)
    for scale in (1.0, math.inf, math.nan, -math.inf, 2.0 ** 127):
        cache.scales[0] = scale
        _check(cached_attention(q, cache, 0, _ints([0, 1], gpu)), o, A, dtype)
