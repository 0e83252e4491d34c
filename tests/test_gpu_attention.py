"""prompt_attention and cached_attention against the definition in 64 bits.

Bar, per element, with u the unit roundoff of the 16-bit type (2^-8 bf16, 2^-11 f16) and A = sum_j w_j |v_j| over the
exact weights w: the kernels round each weight to 16 bits (u A) and the result once (u |o|), and everything
else is fp32: scores below 64 in magnitude carry at most about 2^-17 into the exponent, sums of up to
thousands of terms less, together under 2^-14 A. So |error| <= u (A + |o|) + 2^-14 A, and the smallest value of the
type (subnormal results).
"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _dtype(name):
    import torch
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


def _normal(seed, shape, dtype, dev, scale=1.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(dev)


def _offsets(lens, dev):
    import torch
    return torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).to(dev)


def _rows64(q, k, v, seen, scale):
    """One head in 64 bits: q (n, D), k, v (m, D); row t sees the first seen[t] keys and reads no other.
    Returns o and A."""
    o, A = np.zeros(q.shape), np.zeros(q.shape)
    for t, s in enumerate(seen):
        if s > 0:
            x = (k[:s] @ q[t]) * scale
            w = np.exp(x - x.max())
            w /= w.sum()
            o[t], A[t] = w @ v[:s], w @ np.abs(v[:s])
    return o, A


def _check(got, o, A, dtype):
    u, tiny = (2.0 ** -8, 2.0 ** -133) if dtype == "bf16" else (2.0 ** -11, 2.0 ** -24)
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    bar = u * (A + np.abs(o)) + 2.0 ** -14 * A + tiny
    worst = np.max(np.abs(got - o) - bar)
    assert worst <= 0, worst


def _prompt64(q, k, v, qs, ks, causal, scale):
    q, k, v = (x.double().cpu().numpy() for x in (q, k, v))
    H, G = q.shape[1], q.shape[1] // k.shape[1]
    o, A = np.zeros(q.shape), np.zeros(q.shape)
    a = c = 0
    for n, m in zip(qs, ks):
        seen = [min(max(t + 1 + m - n, 0), m) if causal else m for t in range(n)]
        for h in range(H):
            o[a:a + n, h], A[a:a + n, h] = _rows64(q[a:a + n, h], k[c:c + m, h // G], v[c:c + m, h // G], seen, scale)
        a, c = a + n, c + m
    return o, A


LENGTHS = {
    "one": ([1], None),
    "below a tile": ([37], None),
    "tile edges": ([64, 128, 129, 63, 65, 127], None),
    "empty between": ([0, 5, 0, 0, 200, 1, 0], None),
    "more keys": ([3, 128, 1, 0, 70], [300, 130, 64, 9, 71]),
    "fewer keys, none": ([100, 20, 4, 140], [40, 0, 1, 70]),
}


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(14, 2, 64, "bf16"), (4, 1, 128, "fp16"), (3, 3, 40, "bf16"), (6, 2, 112, "fp16")])
def test_prompt(gpu, lengths, causal, heads, kv, dim, dtype):
    import torch
    from tensorpack_amd.attention import prompt_attention
    print("prompt", lengths, causal, heads, kv, dim, dtype, flush=True)
    qs, ks = LENGTHS[lengths]
    ks = ks or qs
    dt = _dtype(dtype)
    q, k, v = (_normal(s, (n, h, dim), dt, gpu, f) for s, n, h, f in
               ((1, sum(qs), heads, 2.0), (2, sum(ks), kv, 1.0), (3, sum(ks), kv, 1.0)))
    got = prompt_attention(q, k, v, _offsets(qs, gpu), _offsets(ks, gpu), causal=causal)
    assert got.dtype == dt and got.shape == q.shape
    _check(got, *_prompt64(q, k, v, qs, ks, causal, dim ** -0.5), dtype)
    again = prompt_attention(q, k, v, _offsets(qs, gpu), _offsets(ks, gpu), causal=causal)
    assert torch.equal(got, again)


@pytest.mark.parametrize("heads,kv,dim,dtype,causal", [(14, 2, 64, "bf16", True), (4, 4, 128, "fp16", True), (2, 1, 40, "bf16", False)])
@pytest.mark.parametrize("new,keys", [([1], [3000]), ([130], [1500]), ([5, 0, 60, 3], [700, 100, 61, 2500])])
def test_prompt_few_rows_on_many_keys(gpu, new, keys, heads, kv, dim, dtype, causal):
    # keys split over blocks: parts with no keys for some rows, for some waves, for a whole sequence
    import torch
    from tensorpack_amd.attention import prompt_attention
    print("parts", new, keys, heads, kv, dim, dtype, causal, flush=True)
    q, k, v = (_normal(s, (sum(n), h, dim), _dtype(dtype), gpu, f) for s, n, h, f in
               ((1, new, heads, 2.0), (2, keys, kv, 1.0), (3, keys, kv, 1.0)))
    cq, ck = _offsets(new, gpu), _offsets(keys, gpu)
    got = prompt_attention(q, k, v, cq, ck, causal=causal)
    _check(got, *_prompt64(q, k, v, new, keys, causal, dim ** -0.5), dtype)
    assert torch.equal(got, prompt_attention(q, k, v, cq, ck, causal=causal))


def test_prompt_parts_ignore_what_they_do_not_see(gpu):
    import torch
    from tensorpack_amd.attention import prompt_attention
    q, k, v = (_normal(s, (n, 2, 64), _dtype("bf16"), gpu) for s, n in ((1, 50), (2, 2000), (3, 2000)))
    clean = prompt_attention(q, k, v, _offsets([50], gpu), _offsets([2000], gpu)).double().cpu().numpy()
    o, A = _prompt64(q, k, v, [50], [2000], True, 0.125)
    k[1980], v[1980] = math.nan, math.inf
    got = prompt_attention(q, k, v, _offsets([50], gpu), _offsets([2000], gpu))
    _check(got[:30], o[:30], A[:30], "bf16")
    assert torch.isnan(got[30:]).all() and np.isfinite(clean).all()
    v[5] = math.nan                                              # seen by all
    assert torch.isnan(prompt_attention(q, k, v, _offsets([50], gpu), _offsets([2000], gpu))).all()
    few = prompt_attention(q, k[:1030], v[:1030], _offsets([20, 30], gpu), _offsets([1030, 0], gpu))   # a sequence without keys
    assert torch.isnan(few[:20]).all() and not few[20:].any()


def test_prompt_many_sequences(gpu):
    # more sequences than a wave has lanes, tiles of several levels
    from tensorpack_amd.attention import prompt_attention
    rng = np.random.RandomState(5)
    qs = rng.randint(0, 40, size=150).tolist()
    qs[70], qs[149] = 300, 131
    q, k, v = (_normal(s, (sum(qs), h, 64), _dtype("bf16"), gpu) for s, h in ((1, 2), (2, 1), (3, 1)))
    _check(prompt_attention(q, k, v, _offsets(qs, gpu)), *_prompt64(q, k, v, qs, qs, True, 0.125), "bf16")


def test_prompt_strides_and_out(gpu):
    import torch
    from tensorpack_amd.attention import prompt_attention
    n, H, KV, D = 150, 4, 2, 64
    x = _normal(7, (n, (H + 2 * KV) * D), _dtype("bf16"), gpu)
    q, k, v = (t.unflatten(1, (-1, D)) for t in x.split([H * D, KV * D, KV * D], dim=1))
    cu = _offsets([n], gpu)
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu)
    assert torch.equal(prompt_attention(q, k, v, cu), want)                       # rows of one fused product
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(prompt_attention(*heads_first, cu), want)
    odd = torch.empty((n, H * D + 3), dtype=q.dtype, device=gpu)[:, 1:1 + H * D].unflatten(1, (H, D))
    odd.copy_(q)
    assert torch.equal(prompt_attention(odd, k, v, cu), want)                     # unaligned rows: copied
    wide = torch.full((n + 3, 2 * H, D), 7.0, dtype=q.dtype, device=gpu)
    assert prompt_attention(q, k, v, cu, out=wide[2:2 + n, ::2]) is not None
    assert torch.equal(wide[2:2 + n, ::2], want)
    wide[2:2 + n, ::2] = 7.0
    assert torch.equal(wide, torch.full_like(wide, 7.0))                          # nothing else was written
    one = k[:1].expand(n, KV, D)                                                  # a broadcast row
    assert torch.equal(prompt_attention(q, one, v, cu), prompt_attention(q, one.contiguous(), v, cu))


def test_prompt_ignores_what_it_does_not_see(gpu):
    # infinities and NaN in keys and values behind the mask, in other sequences and past the end
    import torch
    from tensorpack_amd.attention import prompt_attention
    qs = [70, 50, 130]
    q, k, v = (_normal(s, (250, h, 64), _dtype("bf16"), gpu) for s, h in ((1, 4), (2, 2), (3, 2)))
    for at, x in ((60, math.nan), (115, math.inf), (240, -math.inf)):
        k[at], v[at] = x, x
    got = prompt_attention(q, k, v, _offsets(qs, gpu)).double().cpu().numpy()
    clean_k, clean_v = k.clone(), v.clone()
    for at in (60, 115, 240):
        clean_k[at], clean_v[at] = 0, 0
    o, A = _prompt64(q, clean_k, clean_v, qs, qs, True, 0.125)
    a = 0
    for n, first in zip(qs, (60, 45, 120)):
        _check(torch.from_numpy(got[a:a + first]), o[a:a + first], A[a:a + first], "bf16")
        assert not np.isfinite(got[a + first:a + n]).any() or first == 120        # an infinite V can be weighed by 0
        a += n


def test_rows_without_keys_beside_a_nan(gpu):
    # rows that see nothing are 0 also where the tile's keys hold a NaN
    import torch
    from tensorpack_amd.attention import cached_attention, prompt_attention
    q, k, v = (_normal(s, (n, 2, 64), _dtype("bf16"), gpu) for s, n in ((1, 100), (2, 40), (3, 40)))
    v[0], k[39] = math.nan, math.nan
    got = prompt_attention(q, k, v, _offsets([100], gpu), _offsets([40], gpu))    # the first 60 queries precede every key
    assert not got[:60].any() and torch.isnan(got[60:]).all()
    v[0] = 0
    assert not torch.isnan(prompt_attention(q, k, v, _offsets([100], gpu), _offsets([40], gpu))[:99]).any()
    cache = _cache(gpu, [70], 16, 1, 64, "bf16", layers=1)
    cache.pool[int(cache.table[0, 0]), 0, 1, :, 3] = math.inf
    q = _normal(9, (1, 8, 2, 64), _dtype("bf16"), gpu)
    got = cached_attention(q, cache, 0, _ints([0], gpu), q_lens=_ints([5], gpu))
    assert not got[0, 5:].any() and not torch.isfinite(got[0, :5]).any()


def test_prompt_all_nan_ends(gpu):
    # every key a NaN: the rows are NaN, without a plain loop over all of them
    import torch
    from tensorpack_amd.attention import prompt_attention
    q, k, v = (_normal(s, (4096, 4, 64), _dtype("bf16"), gpu) for s in (1, 2, 3))
    k[2048:], v[2048:] = math.nan, math.nan
    got = prompt_attention(q, k, v, _offsets([4096], gpu))
    assert torch.isnan(got[2048:]).all() and torch.isfinite(got[:2048]).all()


def test_prompt_large_scores(gpu):
    # one key takes all the weight; scores of the type's range; a scale of its own
    from tensorpack_amd.attention import prompt_attention
    q, k, v = (_normal(s, (200, 2, 64), _dtype("bf16"), gpu, f) for s, f in ((1, 30.0), (2, 30.0), (3, 1.0)))
    got = prompt_attention(q, k, v, _offsets([200], gpu), scale=0.005)
    _check(got, *_prompt64(q, k, v, [200], [200], True, 0.005), "bf16")
    # scores near 10^7: the exponent's own rounding is the same for every key of a row, so it drops out, and keys
    # that are not within 0.3 of the largest weigh less than exp(-30)
    sharp = prompt_attention(q, k, v, _offsets([200], gpu), scale=100.0)
    qq, kk, vv = (x.double().cpu().numpy() for x in (q, k, v))
    for h in range(2):
        s = np.where(np.tril(np.ones((200, 200), bool)), qq[:, h] @ kk[:, h].T, -np.inf)
        top = np.sort(s, axis=1)[:, -2:]
        clear = np.nonzero(top[:, 1] - top[:, 0] > 0.3)[0]
        assert clear.size > 150
        o = vv[s.argmax(1)[clear], h]
        _check(sharp[clear.tolist(), h], o, np.abs(o), "bf16")


def test_prompt_other_stream_and_graph(gpu):
    import torch
    from tensorpack_amd.attention import prompt_attention
    qs = [90, 0, 200]
    q, k, v = (_normal(s, (290, h, 128), _dtype("fp16"), gpu) for s, h in ((1, 4), (2, 4), (3, 4)))
    cu = _offsets(qs, gpu)
    want = prompt_attention(q, k, v, cu)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = prompt_attention(q, k, v, cu)
    st.synchronize()
    assert torch.equal(got, want)
    out, g = torch.empty_like(q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        prompt_attention(q, k, v, cu, out=out)
    for lens in ([90, 0, 200], [10, 200, 80], [290, 0, 0]):                       # lengths stay on the device
        cu.copy_(_offsets(lens, gpu))
        g.replay()
        assert torch.equal(out, prompt_attention(q, k, v, cu))


def test_prompt_bad_offsets_stay_in_bounds(gpu):
    import torch
    from tensorpack_amd.attention import prompt_attention
    q, k, v = (_normal(s, (64, 2, 64), _dtype("bf16"), gpu) for s in (1, 2, 3))
    for cu in ([0, 1000], [-5, 64], [0, 40, 20, 64], [50, 10, 70, -3]):
        out = prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=gpu), out=torch.zeros_like(q))
        assert torch.isfinite(out).all()


def test_prompt_refusals(gpu):
    import torch
    from tensorpack_amd.attention import prompt_attention
    q, k = _normal(1, (8, 4, 64), _dtype("bf16"), gpu), _normal(2, (8, 2, 64), _dtype("bf16"), gpu)
    cu = _offsets([8], gpu)
    bad = [
        (q.float(), k.float(), k.float(), cu, None, {}), (q, k.half(), k.half(), cu, None, {}),
        (q, k, k[:4], cu, None, {}), (q[:, :3], k, k, cu, None, {}), (q, k[:4], k[:4], cu, None, {}),
        (q, k[..., :32], k[..., :32], cu, None, {}), (q, k, k, cu.long(), None, {}), (q, k, k, cu, _offsets([4, 4], gpu), {}),
        (q[..., :12], k[..., :12], k[..., :12], cu, None, {}), (q, k, k, cu, None, {"scale": 0.0}),
        (q, k, k, cu, None, {"scale": math.nan}), (q, k, k, cu, None, {"out": q.float()}), (q, k, k, cu.cpu(), None, {}),
        (q[0], k, k, cu, None, {}),
        (torch.zeros(8, 2, 136, dtype=q.dtype, device=gpu),) * 3 + (cu, None, {}),
    ]
    for q_, k_, v_, c, ck, kw in bad:
        with pytest.raises(ValueError):
            prompt_attention(q_, k_, v_, c, ck, **kw)
    assert prompt_attention(q[:0], k[:0], k[:0], _offsets([0], gpu)).shape == (0, 4, 64)
    assert prompt_attention(q[:0], k[:0], k[:0], _offsets([], gpu)).shape == (0, 4, 64)


# ---- the cache's attention ----
def _cache(dev, lens, page, KV, D, dtype, seed=3, layers=2, extra=5, spread=True, share=None, junk=None):
    """A cache whose sequences hold `lens` tokens in scattered pages; share = (members, tokens): runs of `members`
    sequences hold the same pages for their first `tokens`. Free pages and page ends hold `junk`."""
    import torch
    from tensorpack_amd.cache import PagedCache
    rng = np.random.RandomState(seed)
    need = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(need) + extra).tolist() if spread else list(range(sum(need) + extra))
    table = np.full((len(lens) + 2, max(need + [1]) + 1), -1, np.int32)
    members, common = share or (1, 0)
    for i, n in enumerate(need):
        first = i - i % members
        own = common // page if i != first else 0
        table[i, :own] = table[first, :own]
        for j in range(own, n):
            table[i, j] = ids.pop()
    n_pages = sum(need) + extra
    refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
    pool = _normal(seed, (n_pages, layers, 2, KV, page, D), _dtype(dtype), dev)
    if junk is not None:
        pool[torch.from_numpy(refs == 0).to(dev)] = junk
        for i, n in enumerate(lens):
            if n % page:
                pool[int(table[i, n // page]), :, :, :, n % page:] = junk
    full = np.zeros(len(lens) + 2, np.int32)
    full[:len(lens)] = lens
    up = lambda a: torch.from_numpy(a).to(dev)
    return PagedCache.from_buffers(pool, up(table), up(full), up(refs))


def _cached64(q, cache, layer, seqs, q_lens, scale):
    pool, table, lens = cache.pool.double().cpu().numpy(), cache.table.cpu().numpy(), cache.lens.cpu().numpy()
    q = q.double().cpu().numpy()
    B, T, H, D = q.shape
    G, page = H // cache.n_kv_heads, cache.page_size
    o, A = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        s, ql = seqs[b], T if q_lens is None else q_lens[b]
        at = np.arange(lens[s])
        for h in range(H):
            kv = pool[table[s][at // page], layer, :, h // G, at % page]
            seen = [max(lens[s] - ql + t + 1, 0) if t < ql else 0 for t in range(T)]
            o[b, :, h], A[b, :, h] = _rows64(q[b, :, h], kv[:, 0], kv[:, 1], seen, scale)
    return o, A


def _ints(x, dev):
    import torch
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads,kv,dim,dtype,tokens", [(14, 2, 64, "bf16", 1), (4, 1, 128, "fp16", 3), (3, 3, 40, "bf16", 2),
                                                      (8, 1, 112, "fp16", 8), (16, 2, 128, "bf16", 16)])
def test_cached(gpu, page, heads, kv, dim, dtype, tokens):
    import torch
    from tensorpack_amd.attention import cached_attention
    print("cached", page, heads, kv, dim, dtype, tokens, flush=True)
    lens = [1, 0, 15, 16, 17, 127, 128, 129, 400, 31, 33, 700]
    cache = _cache(gpu, lens, page, kv, dim, dtype, junk=math.nan)
    q = _normal(9, (len(lens), tokens, heads, dim), _dtype(dtype), gpu, 2.0)
    seqs = list(range(len(lens)))[::-1]
    got = cached_attention(q, cache, 1, _ints(seqs, gpu))
    _check(got, *_cached64(q, cache, 1, seqs, None, dim ** -0.5), dtype)
    q_lens = [(3 * i) % (tokens + 1) for i in range(len(lens))]
    got = cached_attention(q, cache, 0, _ints(seqs, gpu), q_lens=_ints(q_lens, gpu), scale=0.2)
    _check(got, *_cached64(q, cache, 0, seqs, q_lens, 0.2), dtype)
    assert torch.equal(got, cached_attention(q, cache, 0, _ints(seqs, gpu), q_lens=_ints(q_lens, gpu), scale=0.2))


def test_cached_long_and_many(gpu):
    # one long sequence cut over many blocks beside many short ones
    from tensorpack_amd.attention import cached_attention
    lens = [20000] + [(37 * i) % 90 for i in range(300)]
    cache = _cache(gpu, lens, 16, 2, 64, "bf16", layers=1)
    q = _normal(9, (len(lens), 1, 4, 64), _dtype("bf16"), gpu, 2.0)
    seqs = list(range(len(lens)))
    _check(cached_attention(q, cache, 0, _ints(seqs, gpu)), *_cached64(q, cache, 0, seqs, None, 0.125), "bf16")


@pytest.mark.parametrize("dim,dtype,heads,kv,tokens,members,common,page", [
    (64, "bf16", 14, 2, 1, 4, 320, 16), (128, "fp16", 8, 2, 3, 3, 256, 64), (128, "bf16", 8, 1, 1, 12, 640, 32),
    (40, "bf16", 2, 2, 1, 2, 16, 16)])
def test_cached_groups(gpu, dim, dtype, heads, kv, tokens, members, common, page):
    from tensorpack_amd.attention import cached_attention
    print("groups", dim, dtype, heads, kv, tokens, members, common, page, flush=True)
    lens = [common + x for x in (1, 40, 3, 200, 16, 17, 129, 90, 33, 300, 5, 64)]
    cache = _cache(gpu, lens, page, kv, dim, dtype, share=(members, common), junk=math.nan)
    q = _normal(9, (12, tokens, heads, dim), _dtype(dtype), gpu, 2.0)
    seqs = list(range(12))
    o, A = _cached64(q, cache, 1, seqs, None, dim ** -0.5)
    groups = list(range(0, 12, members)) + [12]
    call = lambda g, p: cached_attention(q, cache, 1, _ints(seqs, gpu), groups=_ints(g, gpu), prefix_lens=_ints(p, gpu))
    _check(call(groups, [common] * (len(groups) - 1)), o, A, dtype)
    _check(call(groups, [common - 5] * (len(groups) - 1)), o, A, dtype)            # rounded down to whole pages
    _check(call(groups, [0] * (len(groups) - 1)), o, A, dtype)
    _check(call([0, 1, 12], [lens[0], 0]), o, A, dtype)                           # a prefix that is the whole sequence
    _check(call([members, 2 * members], [common]) if members < 12 else call([0, 0, 12], [99, common]), o, A, dtype)


def test_cached_prefix_past_a_draft(gpu):
    # a group whose prefix ends within the drafted tokens: rows that see less than the prefix
    from tensorpack_amd.attention import cached_attention
    lens = [64, 64, 70]
    cache = _cache(gpu, lens, 16, 1, 64, "bf16", share=(3, 64))
    q = _normal(9, (3, 8, 2, 64), _dtype("bf16"), gpu, 2.0)
    got = cached_attention(q, cache, 0, _ints([0, 1, 2], gpu), groups=_ints([0, 3], gpu), prefix_lens=_ints([64], gpu))
    _check(got, *_cached64(q, cache, 0, [0, 1, 2], None, 0.125), "bf16")


def test_cached_drafts_hide_later_ones(gpu):
    # a NaN in a later draft's K and V stays out of the rows before it
    from tensorpack_amd.attention import cached_attention
    cache = _cache(gpu, [100, 40], 16, 1, 64, "bf16", layers=1)
    for s, n in ((0, 100), (1, 40)):
        cache.pool[int(cache.table[s, (n - 1) // 16]), 0, :, :, (n - 1) % 16] = math.nan
    q = _normal(9, (2, 4, 4, 64), _dtype("bf16"), gpu, 2.0)
    got = cached_attention(q, cache, 0, _ints([0, 1], gpu))
    assert not np.isfinite(got[:, 3].double().cpu().numpy()).any()
    cache.lens -= 1
    o, A = _cached64(q[:, :3], cache, 0, [0, 1], None, 0.125)
    _check(got[:, :3], o, A, "bf16")


def test_cached_offsets_past_32_bits(gpu):
    # a pool of 9 GB: the last page's byte offset needs more than 32 bits
    import torch
    from tensorpack_amd.attention import cached_attention
    from tensorpack_amd.cache import PagedCache
    page_bytes = 16 * 2 * 8 * 256 * 128 * 2
    n_pages = (9 << 30) // page_bytes
    cache = PagedCache(n_pages, 16, 8, 128, max_seqs=2, max_pages=2, page_size=256, device=gpu)
    cache.pool[n_pages - 1] = _normal(1, (16, 2, 8, 256, 128), _dtype("bf16"), gpu)
    cache.table[0, 0], cache.lens[0] = n_pages - 1, 250
    q = _normal(9, (1, 1, 8, 128), _dtype("bf16"), gpu, 2.0)
    got = cached_attention(q, cache, 15, _ints([0], gpu))
    kv = cache.pool[n_pages - 1, 15].double().cpu().numpy()
    qq = q.double().cpu().numpy()
    for h in range(8):
        o, A = _rows64(qq[0, :, h], kv[0, h], kv[1, h], [250], 128 ** -0.5)
        _check(got[0, :, h], o, A, "bf16")
    del cache
    torch.cuda.empty_cache()


def test_cached_graph_and_stream(gpu):
    import torch
    from tensorpack_amd.attention import cached_attention
    cache = _cache(gpu, [300, 20, 90], 16, 2, 64, "bf16")
    q, seqs = _normal(9, (3, 2, 4, 64), _dtype("bf16"), gpu), _ints([0, 1, 2], gpu)
    out = torch.empty_like(q)
    cached_attention(q, cache, 0, seqs, out=out)                                  # the workspace exists
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = cached_attention(q, cache, 0, seqs)
    st.synchronize()
    assert torch.equal(other, out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cached_attention(q, cache, 0, seqs, out=out)
    for lens in ([300, 20, 90], [10, 0, 95], [304, 32, 1]):
        cache.lens[:3] = _ints(lens, gpu)
        g.replay()
        assert torch.equal(out, cached_attention(q, cache, 0, seqs))


def test_cached_bad_device_values_stay_in_bounds(gpu):
    import torch
    from tensorpack_amd.attention import cached_attention
    cache = _cache(gpu, [100, 60], 16, 1, 64, "bf16")
    q = _normal(9, (2, 1, 2, 64), _dtype("bf16"), gpu)
    assert not cached_attention(q, cache, 0, _ints([-1, 99], gpu)).any()          # sequences that do not exist
    cache.lens[0], cache.lens[1] = 1 << 30, -7
    cache.table[0] = torch.arange(cache.max_pages, device=gpu) * 1000 - 1
    cached_attention(q, cache, 0, _ints([0, 1], gpu))
    for groups, prefix in (([0, 2], [1 << 30]), ([2, 0], [16]), ([-5, 99], [48])):
        cached_attention(q, cache, 0, _ints([0, 1], gpu), groups=_ints(groups, gpu), prefix_lens=_ints(prefix, gpu))
    torch.cuda.synchronize()


def test_cached_refusals(gpu):
    from tensorpack_amd.attention import cached_attention
    cache = _cache(gpu, [10, 20], 16, 2, 64, "bf16")
    q, seqs = _normal(9, (2, 1, 4, 64), _dtype("bf16"), gpu), _ints([0, 1], gpu)
    bad = [(q.half(), 0, seqs, {}), (q, 2, seqs, {}), (q, -1, seqs, {}), (q, 0, seqs.long(), {}), (q, 0, seqs[:1], {}),
           (q[..., :32], 0, seqs, {}), (q[:, :, :3], 0, seqs, {}), (q.expand(2, 17, 4, 64), 0, seqs, {}), (q[0], 0, seqs, {}),
           (q, 0, seqs, {"groups": _ints([0, 2], gpu)}), (q, 0, seqs, {"scale": -1.0}),
           (q, 0, seqs, {"groups": _ints([0, 2], gpu), "prefix_lens": _ints([16, 16], gpu)}),
           (q, 0, seqs, {"q_lens": _ints([1], gpu)}), (q, 0, seqs, {"out": q.float()})]
    for q_, layer, s, kw in bad:
        with pytest.raises(ValueError):
            cached_attention(q_, cache, layer, s, **kw)
    assert cached_attention(q[:0], cache, 0, seqs[:0]).shape == (0, 1, 4, 64)
