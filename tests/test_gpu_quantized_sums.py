"""cached_attention over a QuantizedCache: the sum of the weights is that of the weights that are multiplied, so that a constant V comes out
as itself, and a NaN in a query stays one whatever its bits. In all three ways through the keys."""

import math

import numpy as np
import pytest

from test_gpu_attention import _dtype, _ints, _normal
from test_gpu_quantized_attention import _cache
from test_gpu_quantized_range import WAYS

pytestmark = pytest.mark.gpu


def _constant(cache, gpu):
    """V is 1 everywhere, in blocks of different steps."""
    import torch
    e = np.random.RandomState(1).randint(-6, -2, size=tuple(cache.scales[:, :, 1].shape))
    cache.scales[:, :, 1] = torch.from_numpy(2.0 ** e.astype(np.float32)).to(cache.scales)
    codes = torch.from_numpy(2.0 ** -e).to(torch.int8).to(gpu)
    cache.codes[:, :, 1] = codes.repeat_interleave(16, dim=-1)[:, :, :, :, None]


@pytest.mark.parametrize("tokens,heads", WAYS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_constant_value_comes_out_as_itself(gpu, dim, dtype, tokens, heads):
    """Exactly: a result off by less than a quarter of a step is rounded to it, 2^-13 (f16, below 1); what is left are fp32 sums over fewer
    than 2^7 steps of 32 keys a wave and their join, at most 2^9 roundings of 2^-24 in either sum: 2^-14."""
    import torch
    from tensorpack_amd.attention import cached_attention
    lens = [3000, 40, 1, 515]
    cache = _cache(gpu, lens, 16, 1, dim, dtype, layers=1, junk=False)
    _constant(cache, gpu)
    q = _normal(9, (4, tokens, heads, dim), _dtype(dtype), gpu, 2.0)
    seen = torch.tensor([[n - tokens + t + 1 > 0 for t in range(tokens)] for n in lens], device=gpu)
    want = seen.to(q.dtype)[:, :, None, None].expand_as(q)
    for scale in (None, 0.003, 1.5):
        assert torch.equal(cached_attention(q, cache, 0, _ints([0, 1, 2, 3], gpu), scale=scale), want), scale
    # weights of 1 (every 16th key) and others that all round the same way: 1/2 (1 + 0.98 2^-11), 11 bits of which are 1/2
    cache.codes[:, :, 0] = 0
    cache.scales[:, :, 0] = 1.0
    cache.codes[:, :, 0, ..., 0] = -1
    cache.codes[:, :, 0, :, 0, 0] = 0
    q.zero_()
    q[..., 0] = 1
    for share in (0.98, -0.98 / 2, 0.49):
        got = cached_attention(q, cache, 0, _ints([0, 1, 2, 3], gpu), scale=-math.log(0.5 * (1 + share * 2.0 ** -11)))
        assert torch.equal(got, want), (share, float((got.float() - want.float()).abs().max()))


@pytest.mark.parametrize("tokens,heads", WAYS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_nan_of_any_bits(gpu, dtype, tokens, heads):
    import torch
    from tensorpack_amd.attention import cached_attention
    cache = _cache(gpu, [100, 300], 16, 1, 64, dtype, layers=1)
    first = 0x7F81 if dtype == "bf16" else 0x7C01
    for bits in (first, 0x7FFF, first | 0x8000, 0xFFFF):
        q = _normal(9, (2, tokens, heads, 64), _dtype(dtype), gpu, 2.0)
        clean = cached_attention(q, cache, 0, _ints([0, 1], gpu))
        q.view(torch.int16)[1, tokens - 1, 2, 7] = bits - (bits & 0x8000) * 2
        got = cached_attention(q, cache, 0, _ints([0, 1], gpu))
        assert torch.isnan(q[1, tokens - 1, 2, 7]) and torch.isnan(got[1, tokens - 1, 2]).all(), hex(bits)
        got[1, tokens - 1, 2] = clean[1, tokens - 1, 2]
        assert torch.equal(got, clean)
