"""Views that torch calls contiguous though the kernels cannot read them in place: a start off a 16-byte boundary, one row of
a wider tensor. Equality with the same values in memory of their own."""

import pytest

pytestmark = pytest.mark.gpu


def _ints(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _normal(dev, seed, *shape, dtype=None):
    import torch
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed))
    return x.to(dev, dtype or torch.bfloat16)


def _offset(x):
    """x's values, contiguous, one element past an aligned start."""
    import torch
    y = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
    y.copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16
    return y


def _one_row(x):
    """x's values (a single row) as a view into a row of odd width."""
    import torch
    assert x.shape[0] == 1
    n = x[0].numel()
    y = torch.empty(n + 3, dtype=x.dtype, device=x.device).as_strided(x.shape, (n + 3,) + x.stride()[1:])
    y.copy_(x)
    assert y.is_contiguous() and y.stride(0) % 4
    return y


@pytest.mark.parametrize("view,rows", [(_offset, 1), (_offset, 37), (_one_row, 1)])
def test_prompt(gpu, view, rows):
    import torch
    from tensorpack_amd.attention import prompt_attention
    q, k, v = _normal(gpu, 1, rows, 4, 64), _normal(gpu, 2, rows, 2, 64), _normal(gpu, 3, rows, 2, 64)
    cu = _ints([0, rows], gpu)
    want = prompt_attention(q, k, v, cu)
    for i in range(3):
        x = [q, k, v]
        x[i] = view(x[i])
        assert torch.equal(prompt_attention(*x, cu), want), i
    with pytest.raises(ValueError):
        prompt_attention(q, k, v, cu, out=view(q))


@pytest.mark.parametrize("view,seqs,tokens", [(_offset, 2, 3), (_offset, 1, 1), (_one_row, 1, 1), (_one_row, 1, 5)])
def test_cached(gpu, view, seqs, tokens):
    import torch
    from tensorpack_amd.attention import cached_attention
    from tensorpack_amd.cache import PagedCache
    cache = PagedCache(10, 1, 2, 64, max_seqs=2, max_pages=5, device=gpu)
    cache.pool.copy_(_normal(gpu, 1, *cache.pool.shape))
    ids = _ints(list(range(seqs)), gpu)
    cache.extend(ids, _ints([40] * seqs, gpu))
    q = _normal(gpu, 2, seqs, tokens, 4, 64)
    assert torch.equal(cached_attention(view(q), cache, 0, ids), cached_attention(q, cache, 0, ids))


@pytest.mark.parametrize("view,rows", [(_offset, 1), (_offset, 21), (_one_row, 1)])
@pytest.mark.parametrize("fp32", [False, True])
def test_append(gpu, view, rows, fp32):
    import torch
    from tensorpack_amd.cache import PagedCache
    dt = torch.float32 if fp32 else torch.bfloat16
    k, v = _normal(gpu, 1, rows, 2, 64, dtype=dt), _normal(gpu, 2, rows, 2, 64, dtype=dt)
    pools = []
    for f in (lambda x: x, view):
        cache = PagedCache(4, 1, 2, 64, max_seqs=1, max_pages=4, device=gpu)
        cache.pool.zero_()
        cache.extend(_ints([0], gpu), _ints([rows], gpu))
        cache.append(0, f(k), f(v), _ints([0], gpu), _ints([0, rows], gpu))
        pools.append(cache.pool)
    assert torch.equal(*pools) and pools[0].any()
