"""cached_attention over a QuantizedCache against the definition in 64 bits, on the values that its codes stand for.

The bar is that of the 16-bit cache: codes become numbers of the 16-bit type exactly, and what follows rounds each weight
and the result once (see test_gpu_attention)."""

import math

import numpy as np
import pytest

from test_gpu_attention import _check, _dtype, _ints, _normal, _rows64

pytestmark = pytest.mark.gpu


def _cache(dev, lens, page, KV, D, dtype, seed=3, layers=2, extra=5, share=None, exps=(-7, -5), junk=True):
    """A QuantizedCache whose sequences hold `lens` tokens in scattered pages; share = (members, tokens): runs of `members`
    sequences hold the same pages for their first `tokens`. Codes and scales are random; scales of blocks that hold no token are
    anything (NaN, infinities, negative ones, 2 ** 127)."""
    import torch
    from tensorpack_amd.cache import QuantizedCache
    rng = np.random.RandomState(seed)
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + extra
    ids = rng.permutation(n_pages).tolist()
    table = np.full((len(lens) + 2, max(need + [1]) + 1), -1, np.int32)
    members, common = share or (1, 0)
    for i, n in enumerate(need):
        first = i - i % members
        own = common // page if i != first else 0
        table[i, :own] = table[first, :own]
        for j in range(own, n):
            table[i, j] = ids.pop()
    refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
    full = np.zeros(len(lens) + 2, np.int32)
    full[:len(lens)] = lens
    room = -(-D // 16) * 16
    codes_bytes, scales_bytes = 2 * layers * KV * page * room, 4 * layers * KV * (page // 16)
    pool = torch.from_numpy(rng.randint(-128, 128, size=(n_pages, -(-(codes_bytes + scales_bytes) // 16) * 16)).astype(np.int8)).to(dev)
    up = lambda a: torch.from_numpy(a).to(dev)
    c = QuantizedCache.from_buffers(pool, up(table), up(full), up(refs), n_layers=layers, n_kv_heads=KV, head_dim=D, page_size=page,
                                    dtype=_dtype(dtype))
    c.codes.clamp_(min=-127)
    scales = 2.0 ** rng.randint(exps[0], exps[1] + 1, size=tuple(c.scales.shape)).astype(np.float32)
    if junk:
        held = np.zeros((n_pages, page // 16), bool)
        for i, n in enumerate(lens):
            for b in range(-(-n // 16)):
                held[table[i, 16 * b // page], b % (page // 16)] = True
        wild = rng.choice(np.array([math.nan, math.inf, -math.inf, -1.0, 2.0 ** 127, 0.0], np.float32), size=scales.shape)
        scales = np.where(held[:, None, None, None, :], scales, wild)
    c.scales.copy_(torch.from_numpy(scales))
    return c


def _cached64(q, cache, layer, seqs, q_lens, scale):
    codes, scales = cache.codes[:, layer].cpu().numpy(), cache.scales[:, layer].double().cpu().numpy()
    table, lens = cache.table.cpu().numpy(), cache.lens.cpu().numpy()
    q = q.double().cpu().numpy()
    B, T, H, D = q.shape
    G, page = H // cache.n_kv_heads, cache.page_size
    o, A = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        s, ql = seqs[b], T if q_lens is None else q_lens[b]
        at = np.arange(lens[s])
        p = table[s][at // page]
        for h in range(H):
            k, v = (codes[p, j, h // G, at % page] * scales[p, j, h // G, at % page // 16][:, None] for j in (0, 1))
            seen = [max(lens[s] - ql + t + 1, 0) if t < ql else 0 for t in range(T)]
            o[b, :, h], A[b, :, h] = _rows64(q[b, :, h], k, v, seen, scale)
    return o, A


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads,kv,dim,dtype,tokens", [(14, 2, 64, "bf16", 1), (4, 1, 128, "fp16", 3), (3, 3, 40, "bf16", 2), (24, 1, 16, "fp16", 1),
                                                      (8, 1, 112, "fp16", 8), (16, 2, 128, "bf16", 16), (2, 1, 8, "bf16", 5)])
def test_lengths_and_heads(gpu, page, heads, kv, dim, dtype, tokens):
    import torch
    from tensorpack_amd.attention import cached_attention
    print("codes", page, heads, kv, dim, dtype, tokens, flush=True)
    lens = [1, 0, 15, 16, 17, 127, 128, 129, 400, 31, 33, 700, 63, 64, 65]
    cache = _cache(gpu, lens, page, kv, dim, dtype)
    q = _normal(9, (len(lens), tokens, heads, dim), _dtype(dtype), gpu, 2.0)
    seqs = list(range(len(lens)))[::-1]
    got = cached_attention(q, cache, 1, _ints(seqs, gpu))
    _check(got, *_cached64(q, cache, 1, seqs, None, dim ** -0.5), dtype)
    q_lens = [(3 * i) % (tokens + 1) for i in range(len(lens))]
    got = cached_attention(q, cache, 0, _ints(seqs, gpu), q_lens=_ints(q_lens, gpu), scale=0.2 if dim > 16 else 0.5)
    _check(got, *_cached64(q, cache, 0, seqs, q_lens, 0.2 if dim > 16 else 0.5), dtype)
    assert torch.equal(got, cached_attention(q, cache, 0, _ints(seqs, gpu), q_lens=_ints(q_lens, gpu), scale=0.2 if dim > 16 else 0.5))


@pytest.mark.parametrize("heads,dim", [(4, 64), (2, 128)])
def test_long_and_many(gpu, heads, dim):
    # one long sequence cut over many blocks beside many short ones
    from tensorpack_amd.attention import cached_attention
    lens = [20000] + [(37 * i) % 90 for i in range(300)]
    cache = _cache(gpu, lens, 16, 2, dim, "bf16", layers=1)
    q = _normal(9, (len(lens), 1, heads, dim), _dtype("bf16"), gpu, 2.0)
    seqs = list(range(len(lens)))
    _check(cached_attention(q, cache, 0, _ints(seqs, gpu)), *_cached64(q, cache, 0, seqs, None, dim ** -0.5), "bf16")


@pytest.mark.parametrize("dim,dtype,heads,kv,tokens,members,common,page", [
    (64, "bf16", 14, 2, 1, 4, 320, 16), (128, "fp16", 8, 2, 3, 3, 256, 64), (128, "bf16", 8, 1, 1, 12, 640, 32), (40, "bf16", 2, 2, 1, 2, 16, 16),
    (64, "fp16", 8, 1, 5, 6, 1024, 128)])
def test_groups(gpu, dim, dtype, heads, kv, tokens, members, common, page):
    from tensorpack_amd.attention import cached_attention
    print("groups", dim, dtype, heads, kv, tokens, members, common, page, flush=True)
    lens = [common + x for x in (1, 40, 3, 200, 16, 17, 129, 90, 33, 300, 5, 64)]
    cache = _cache(gpu, lens, page, kv, dim, dtype, share=(members, common))
    q = _normal(9, (12, tokens, heads, dim), _dtype(dtype), gpu, 2.0)
    seqs = list(range(12))
    o, A = _cached64(q, cache, 1, seqs, None, dim ** -0.5)
    groups = list(range(0, 12, members)) + [12]
    call = lambda g, p: cached_attention(q, cache, 1, _ints(seqs, gpu), groups=_ints(g, gpu), prefix_lens=_ints(p, gpu))
    _check(call(groups, [common] * (len(groups) - 1)), o, A, dtype)
    _check(call(groups, [common - 5] * (len(groups) - 1)), o, A, dtype)            # rounded down to whole pages
    _check(call(groups, [0] * (len(groups) - 1)), o, A, dtype)
    _check(call([0, 1, 12], [lens[0], 0]), o, A, dtype)                           # a prefix that is the whole sequence


def test_prefix_past_a_draft(gpu):
    from tensorpack_amd.attention import cached_attention
    lens = [64, 64, 70]
    cache = _cache(gpu, lens, 16, 1, 64, "bf16", share=(3, 64))
    q = _normal(9, (3, 8, 2, 64), _dtype("bf16"), gpu, 2.0)
    got = cached_attention(q, cache, 0, _ints([0, 1, 2], gpu), groups=_ints([0, 3], gpu), prefix_lens=_ints([64], gpu))
    _check(got, *_cached64(q, cache, 0, [0, 1, 2], None, 0.125), "bf16")


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("fp16", 128), ("bf16", 128)])
def test_scales_far_apart(gpu, dtype, dim):
    """Blocks whose scales are at both ends of the range: V's enter the result as they are, a block of tiny ones still has its
    keys' weights. (K's scales stay moderate: scores below 64.)"""
    import torch
    from tensorpack_amd.attention import cached_attention
    lo, hi = {"bf16": (-100, 100), "fp16": (-24, 8)}[dtype]
    lens = [500, 17, 40]
    cache = _cache(gpu, lens, 16, 1, dim, dtype, layers=1)
    rng = np.random.RandomState(4)
    v = 2.0 ** rng.choice([lo, lo, lo + 1, -6, -6, 0], size=tuple(cache.scales[:, :, 1].shape)).astype(np.float32)
    q = _normal(9, (3, 1, 4, dim), _dtype(dtype), gpu, 2.0)
    for high in (False, True):
        if high:
            v[int(cache.table[0, 20])] = 2.0 ** hi
        cache.scales[:, :, 1] = torch.from_numpy(v).to(cache.scales)
        _check(cached_attention(q, cache, 0, _ints([0, 1, 2], gpu)), *_cached64(q, cache, 0, [0, 1, 2], None, dim ** -0.5), dtype)


def test_infinite_and_nan_queries_stay_in_their_rows(gpu):
    import torch
    from tensorpack_amd.attention import cached_attention
    cache = _cache(gpu, [100, 300], 16, 2, 64, "bf16")
    for heads, tokens in ((4, 1), (8, 6), (32, 8)):
        q = _normal(9, (2, tokens, heads, 64), _dtype("bf16"), gpu, 2.0)
        clean = cached_attention(q, cache, 0, _ints([0, 1], gpu))
        q[0, 0, 1, 5], q[1, tokens - 1, 2, 0] = math.nan, math.inf
        got = cached_attention(q, cache, 0, _ints([0, 1], gpu))
        touched = torch.zeros(got.shape[:3], dtype=torch.bool, device=gpu)
        touched[0, 0, 1] = touched[1, tokens - 1, 2] = True
        assert torch.isnan(got[0, 0, 1]).all() and torch.equal(got[~touched], clean[~touched])


def test_offsets_past_32_bits(gpu):
    # a pool of 9 GB: the last page's byte offset needs more than 32 bits
    import torch
    from tensorpack_amd.attention import cached_attention
    from tensorpack_amd.cache import QuantizedCache
    one = QuantizedCache(1, 16, 8, 128, max_seqs=2, max_pages=2, page_size=256, device=gpu)
    n_pages = (9 << 30) // one.pool.shape[1]
    cache = QuantizedCache(n_pages, 16, 8, 128, max_seqs=2, max_pages=2, page_size=256, device=gpu)
    cache.table[0, 0], cache.lens[0], cache.refs[n_pages - 1] = n_pages - 1, 250, 1
    k, v = (_normal(s, (250, 8, 128), _dtype("bf16"), gpu) for s in (1, 2))
    cache.append(15, k, v, _ints([0], gpu), _ints([0, 250], gpu))
    cache.check()
    kv = [x.double().cpu().numpy() for x in cache.read(15, _ints([0], gpu), _ints([0, 250], gpu), 250)]
    assert np.abs(kv[0] - k.double().cpu().numpy()).max() < 0.05
    q = _normal(9, (1, 1, 8, 128), _dtype("bf16"), gpu, 2.0)
    got = cached_attention(q, cache, 15, _ints([0], gpu))
    qq = q.double().cpu().numpy()
    for h in range(8):
        o, A = _rows64(qq[0, :, h], kv[0][:, h], kv[1][:, h], [250], 128 ** -0.5)
        _check(got[0, :, h], o, A, "bf16")
    del cache
    torch.cuda.empty_cache()


def test_graph_and_stream(gpu):
    import torch
    from tensorpack_amd.attention import cached_attention
    cache = _cache(gpu, [300, 20, 90], 16, 2, 64, "bf16")
    q, seqs = _normal(9, (3, 2, 4, 64), _dtype("bf16"), gpu), _ints([0, 1, 2], gpu)
    out = torch.empty_like(q)
    cached_attention(q, cache, 0, seqs, out=out)
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
    own = q.clone()
    assert torch.equal(cached_attention(own, cache, 0, seqs, out=own), out)        # into its own queries


def test_bad_device_values_stay_in_bounds(gpu):
    import torch
    from tensorpack_amd.attention import cached_attention
    cache = _cache(gpu, [100, 60], 16, 1, 64, "bf16")
    q = _normal(9, (2, 1, 2, 64), _dtype("bf16"), gpu)
    assert not cached_attention(q, cache, 0, _ints([-1, 99], gpu)).any()          # sequences that do not exist
    cache.lens[0], cache.lens[1] = 1 << 30, -7
    cache.table[0] = torch.arange(cache.max_pages, device=gpu) * 1000 - 1
    assert torch.isfinite(cached_attention(q, cache, 0, _ints([0, 1], gpu))).all()
    for groups, prefix in (([0, 2], [1 << 30]), ([2, 0], [16]), ([-5, 99], [48])):
        cached_attention(q, cache, 0, _ints([0, 1], gpu), groups=_ints(groups, gpu), prefix_lens=_ints(prefix, gpu))
    cache.append(0, q[0].expand(4, 2, 64)[:, :1], q[0].expand(4, 2, 64)[:, :1], _ints([0, 1], gpu), _ints([0, 2, 4], gpu))
    cache.read(0, _ints([0, 1], gpu), _ints([0, 50, 100], gpu), 100)
    torch.cuda.synchronize()


@pytest.mark.parametrize("tokens,heads", [(1, 8), (4, 8), (12, 16)])
def test_runs_of_many_pages(gpu, tokens, heads):
    """Single keys' runs over more pages than a wave keeps at hand (64), in all three ways through the keys."""
    from tensorpack_amd.attention import cached_attention
    lens = [9000, 4100, 2050]
    cache = _cache(gpu, lens, 16, 1, 64, "bf16", layers=1)
    q = _normal(9, (3, tokens, heads, 64), _dtype("bf16"), gpu, 2.0)
    rows = [0, 1, heads - 1]
    got = cached_attention(q, cache, 0, _ints([0, 1, 2], gpu))
    _check(got[:, :, rows], *_cached64(q[:, :, rows], cache, 0, [0, 1, 2], None, 0.125), "bf16")


def test_batches_beyond_the_lists_in_lds(gpu):
    """600 sequences, prefixes of 60 groups, in any order of the cache's rows."""
    from tensorpack_amd.attention import cached_attention
    lens = [64 + i % 7 for i in range(600)]
    cache = _cache(gpu, lens, 16, 1, 64, "fp16", layers=1, share=(10, 64))
    q = _normal(9, (600, 1, 4, 64), _dtype("fp16"), gpu, 2.0)
    seqs = list(range(600))
    got = cached_attention(q, cache, 0, _ints(seqs, gpu), groups=_ints(list(range(0, 601, 10)), gpu), prefix_lens=_ints([64] * 60, gpu))
    _check(got, *_cached64(q, cache, 0, seqs, None, 0.125), "fp16")


def test_chunks_of_a_prompt(gpu):
    """A prompt fed in pieces of more tokens than cached_attention takes: written, read back, and prompt_attention over all of it."""
    import torch
    from tensorpack_amd.attention import cached_attention, prompt_attention
    from tensorpack_amd.cache import QuantizedCache
    from test_gpu_attention import _prompt64
    cache = QuantizedCache(40, 1, 2, 64, max_seqs=2, max_pages=20, device=gpu)
    k, v = (_normal(s, (230, 2, 64), _dtype("bf16"), gpu) for s in (1, 2))
    q = _normal(3, (230, 8, 64), _dtype("bf16"), gpu, 2.0)
    seq, at = _ints([1], gpu), 0
    for n in (100, 37, 93):
        cache.extend(seq, _ints([n], gpu))
        cache.append(0, k[at:at + n], v[at:at + n], seq, _ints([0, n], gpu))
        at += n
        ck = _ints([0, at], gpu)
        kk, vv = cache.read(0, seq, ck, at)
        got = prompt_attention(q[at - n:at], kk, vv, _ints([0, n], gpu), ck)
        _check(got, *_prompt64(q[at - n:at], kk, vv, [n], [at], True, 0.125), "bf16")
        few = cached_attention(q[at - 4:at][None], cache, 0, seq)
        _check(few[0], *_prompt64(q[at - 4:at], kk, vv, [4], [at], True, 0.125), "bf16")
    cache.check()


def test_refusals(gpu):
    import torch
    from tensorpack_amd.attention import cached_attention
    cache = _cache(gpu, [10, 20], 16, 2, 64, "bf16")
    q, seqs = _normal(9, (2, 1, 4, 64), _dtype("bf16"), gpu), _ints([0, 1], gpu)
    for q_, layer, s, kw in [(q.half(), 0, seqs, {}), (q.to(torch.int8), 0, seqs, {}), (q, 2, seqs, {}), (q, 0, seqs.long(), {}), (q[..., :32], 0, seqs, {}),
                             (q[:, :, :3], 0, seqs, {}), (q.expand(2, 17, 4, 64), 0, seqs, {}), (q, 0, seqs, {"groups": _ints([0, 2], gpu)}),
                             (q, 0, seqs, {"scale": -1.0}), (q, 0, seqs, {"out": q.float()})]:
        with pytest.raises(ValueError):
            cached_attention(q_, cache, layer, s, **kw)
