"""cached_attention over a QuantizedCache at the ends of what its scales, its queries and its table may hold, against the definition in
64 bits with the bar of test_gpu_attention. Each in all three ways through the keys: up to 16 rows, up to 32, and more."""

import math

import numpy as np
import pytest

from test_gpu_attention import _check, _dtype, _ints, _normal, _rows64
from test_gpu_quantized_attention import _cache, _cached64

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


def _check_few(got, q, cache, tokens, heads, scale):
    """_check of layer 0, K/V head 0, with what few rows of bf16 may lose besides: q goes to f16, its largest element scaled to 2^15 or more, so that each of
    them is off by at most half of f16's smallest step, 2^-25, or 2^-40 of the row's largest, and a score by d = scale 2^-40 max |q|
    max over keys of sum |k|. Weights then lie within exp(+-2 d) of theirs, and the result within (exp(2 d) - 1) A."""
    seqs = list(range(q.shape[0]))
    o, A = _cached64(q, cache, 0, seqs, None, scale)
    few = tokens * heads <= 32
    codes, scales = np.abs(cache.codes[:, 0, 0, 0].cpu().numpy().astype(np.float64)), cache.scales[:, 0, 0, 0].double().cpu().numpy()
    table, page = cache.table.cpu().numpy(), cache.page_size
    for b in seqs:
        at = np.arange(int(cache.lens[b]))
        k = codes[table[b][at // page], at % page].sum(-1) * scales[table[b][at // page], at % page // 16]
        d = scale * 2.0 ** -40 * np.abs(q[b].double().cpu().numpy()).max(-1) * k.max() * few
        x = got[b].double().cpu().numpy()
        assert np.isfinite(x).all()
        bar = 2.0 ** -8 * (A[b] + np.abs(o[b])) + (2.0 ** -14 + np.expm1(2 * np.minimum(d, 50.0)))[..., None] * A[b] + 2.0 ** -133
        worst = np.max(np.abs(x - o[b]) - bar)
        assert worst <= 0, (b, worst)


@pytest.mark.parametrize("tokens,heads", WAYS)
def test_queries_of_any_size(gpu, tokens, heads):
    """bf16: rows whose largest element is near the type's largest, or near 2 ** -110, beside keys with the smallest step, or with codes of 0
    and the largest. Scores stay moderate: the large element meets codes of 0, the others are of 2 ** 100 and meet 2 ** -100."""
    import torch
    from tensorpack_amd.attention import cached_attention
    lens = [300, 65, 16]
    cache = _cache(gpu, lens, 16, 1, 64, "bf16", layers=1, exps=(-100, -99), junk=False)
    cache.codes[:, :, 0, ..., 5] = 0
    cache.scales[:, :, 1] = 2.0 ** -6
    for s, block in ((0, 1), (0, 7), (1, 4)):
        page = int(cache.table[s, block])
        cache.codes[page, :, 0] = 0
        cache.scales[page, :, 0] = 2.0 ** 100
    q = _normal(9, (3, tokens, heads, 64), torch.float32, gpu, 2.0 ** -4).double() * 2.0 ** 100
    large = [2.0 ** 114, 2.0 ** 115, -2.0 ** 116, 2.0 ** 120, -2.0 ** 127, 3.38e38, 2.0 ** 101, 2.0 ** 113]
    q[..., 5] = torch.tensor(large, dtype=torch.float64, device=gpu)
    q[1, :, 3] *= 2.0 ** -227                                       # (the row of 2 ** 120: -> 2 ** -107)
    q[2, :, 4] = 0
    q = q.to(torch.float32).bfloat16()
    _check_few(cached_attention(q, cache, 0, _ints([0, 1, 2], gpu)), q, cache, tokens, heads, 0.125)


@pytest.mark.parametrize("tokens,heads", WAYS)
def test_small_queries_on_large_steps(gpu, tokens, heads):
    import torch
    from tensorpack_amd.attention import cached_attention
    lens = [300, 65, 16]
    cache = _cache(gpu, lens, 16, 1, 64, "bf16", layers=1, exps=(99, 100), junk=False)
    cache.scales[:, :, 1] = 2.0 ** -6
    q = (_normal(9, (3, tokens, heads, 64), torch.float32, gpu, 2.0 ** -4).double() * 2.0 ** -100).to(torch.float32).bfloat16()
    _check_few(cached_attention(q, cache, 0, _ints([0, 1, 2], gpu)), q, cache, tokens, heads, 0.125)
