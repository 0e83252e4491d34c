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


@pytest.mark.parametrize("rows,keys", [(150, 150), (50, 2000)])   # keys of a tile by one block, and split over blocks
def test_prompt_into_its_own_queries(gpu, rows, keys):
    """Rows whose unseen keys hold an infinity are computed again from q, which out may be."""
    import torch
    from tensorpack_amd.attention import prompt_attention
    x = _normal(gpu, 1, rows, 2 * 4 * 64)
    k, v = _normal(gpu, 2, keys, 2, 64), _normal(gpu, 3, keys, 2, 64)
    v[keys - 20], v[keys - 3, 1] = float("inf"), float("nan")
    q = x[:, 64:320].unflatten(1, (4, 64))
    cu, ck = _ints([0, rows], gpu), _ints([0, keys], gpu)
    want = prompt_attention(q, k, v, cu, ck)
    assert torch.isfinite(want[:rows - 20]).all() and not torch.isfinite(want[-1]).any()
    bits, around = want.view(torch.int16).clone(), x.clone()
    assert prompt_attention(q, k, v, cu, ck, out=q) is q
    assert torch.equal(q.contiguous().view(torch.int16), bits)
    assert torch.equal(x[:, :64], around[:, :64]) and torch.equal(x[:, 320:], around[:, 320:])


def test_prompt_refuses_its_keys_or_values_as_out(gpu):
    import torch
    from tensorpack_amd.attention import prompt_attention
    q, k, v = (_normal(gpu, s, 9, 2, 64) for s in (1, 2, 3))
    for out in (k, v):
        with pytest.raises(ValueError):
            prompt_attention(q, k, v, _ints([0, 9], gpu), out=out)
    empty = q[:0]
    assert prompt_attention(empty, empty, empty, _ints([0, 0], gpu), out=empty).shape == (0, 2, 64)


def test_cached_into_its_own_queries(gpu):
    import torch
    from tensorpack_amd.attention import cached_attention
    from tensorpack_amd.cache import PagedCache
    cache = PagedCache(10, 1, 2, 64, max_seqs=2, max_pages=5, device=gpu)
    cache.pool.copy_(_normal(gpu, 1, *cache.pool.shape))
    ids = _ints([0, 1], gpu)
    cache.extend(ids, _ints([40, 70], gpu))
    cache.pool[int(cache.table[1, 4]), 0, 1, :, 5] = float("inf")        # the last token of sequence 1
    q = _normal(gpu, 2, 2, 4, 4, 64)
    want = cached_attention(q, cache, 0, ids)
    assert torch.isfinite(want[0]).all() and torch.isfinite(want[1, :3]).all() and not torch.isfinite(want[1, 3]).any()
    assert cached_attention(q, cache, 0, ids, out=q) is q
    assert torch.equal(q.view(torch.int16), want.view(torch.int16))
