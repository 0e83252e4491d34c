"""How far values of a QuantizedCache are off when a block grows token by token, and what a dropped token leaves behind. Bounds: half a step of
each exponent that the block had since the value was written. These double at least, so all together are less than one step of the last."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _ints(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("growth", [0.0, 0.15, 1.0, -0.3])
def test_token_by_token(gpu, dtype, growth):
    """40 tokens one after another, each 2 ** growth times the size of the one before."""
    import torch
    from tensorpack_amd.cache import QuantizedCache
    n, heads, dim = 40, 3, 40
    cache = QuantizedCache(8, 1, heads, dim, max_seqs=1, max_pages=4, dtype=getattr(torch, dtype), device=gpu)
    g = torch.Generator().manual_seed(3)
    x = torch.randn((2, n, heads, dim), generator=g) * 2.0 ** (growth * (torch.arange(n) - n / 2.0) * (0.6 if growth == 1.0 else 1.0))[None, :, None, None]
    x = x.to(getattr(torch, dtype)).to(gpu)
    seq, one, two = _ints([0], gpu), _ints([1], gpu), _ints([0, 1], gpu)
    bound, last, written = np.zeros((2, n, heads)), np.full((2, heads), -1000), np.zeros((2, n, heads))
    for t in range(n):
        cache.extend(seq, one)
        cache.append(0, x[0, t:t + 1], x[1, t:t + 1], seq, two)
        page = int(cache.table[0, t // 16])
        e = np.log2(cache.scales[page, 0, :, :, 0].double().cpu().numpy())
        if t % 16 == 0:
            last[:] = -1000
        assert (e >= last).all()
        first = t // 16 * 16
        bound[:, first:t] += np.where(e > last, 2.0 ** (e - 1), 0.0)[:, None]
        bound[:, t] = 2.0 ** (e - 1)
        written[:, first:t + 1] = 2.0 ** e[:, None]
        last = e
    cache.check()
    got = torch.stack(cache.read(0, seq, _ints([0, n], gpu), n, dtype=torch.float32)).double().cpu().numpy()
    err = np.abs(got - x.double().cpu().numpy())
    assert (err <= bound[..., None]).all()
    assert (bound < written).all() and (err < written[..., None]).all()
    if growth == 1.0:
        assert (err > 0.5 * written[..., None]).any()               # a half step is not the bound
    top = np.abs(x.double().cpu().numpy()).max(-1)
    if growth <= 0:                                                 # nothing larger came: half a step, 1 / 127 of the block's largest
        for a in range(0, n, 16):
            largest = top[:, a:a + 16].max(1)[:, None, :, None]
            if growth < 0:
                assert (err[:, a:a + 1] <= largest / 127).all()
            assert (err[:, a:a + 16] <= 2 * largest / 127).all()


@pytest.mark.parametrize("how", ["truncate", "restore"])
def test_a_dropped_token_leaves_its_step(gpu, how):
    import torch
    from tensorpack_amd.cache import QuantizedCache
    heads, dim = 2, 64
    cache = QuantizedCache(8, 1, heads, dim, max_seqs=1, max_pages=4, device=gpu)
    g = torch.Generator().manual_seed(4)
    k = torch.randn((20, heads, dim), generator=g).bfloat16().to(gpu)
    seq = _ints([0], gpu)
    put = lambda x: (cache.extend(seq, _ints([len(x)], gpu)), cache.append(0, x, x, seq, _ints([0, len(x)], gpu)))
    read = lambda n: torch.stack(cache.read(0, seq, _ints([0, n], gpu), n)).double()
    put(k[:5])
    fine, step = read(5), cache.scales[int(cache.table[0, 0]), 0].clone()
    snapshot = cache.snapshot()
    put(k[5:6] * 64)
    coarse = read(6)[:, :5]
    large = cache.scales[int(cache.table[0, 0]), 0].clone()
    assert (large >= 16 * step).all() and not torch.equal(coarse, fine)
    cache.restore(snapshot) if how == "restore" else cache.truncate(seq, _ints([5], gpu))
    assert torch.equal(read(5), coarse)                             # as the dropped token made them
    assert ((coarse - k[:5].double()).abs() < large.double().amax(-1)[:, None, :, None]).all()
    put(k[5:9])
    assert torch.equal(cache.scales[int(cache.table[0, 0]), 0], large)
    assert torch.equal(read(9)[:, :5], coarse)
    assert ((read(9)[:, 5:] - k[5:9].double()).abs() <= large.double().amax(-1)[:, None, :, None] / 2).all()
    cache.truncate(seq, _ints([0], gpu))
    put(k[:5])
    assert torch.equal(read(5), fine)                               # a block's first token begins anew
