"""Sizes at which the serving kernels change their way: runs of more pages than a wave holds at once, more sequences than
the lists kept in LDS, vocabularies that a block takes in two rounds.

Attention's bar, per element, with u = 2^-8 (bf16), A = sum_j w_j |v_j|: each weight and the result are rounded once, the rest
is fp32: u (A + |o|) + 2^-14 A. Scores stay below 64, sums below 2^17 terms."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _ints(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cache(dev, lens, kv, dim, page=16, seed=3):
    """Sequences of `lens` tokens in scattered pages."""
    import torch
    from tensorpack_amd.cache import PagedCache
    need = [-(-n // page) for n in lens]
    c = PagedCache(sum(need) + 3, 1, kv, dim, max_seqs=len(lens), max_pages=max(need), page_size=page, device=dev)
    g = torch.Generator(device=dev).manual_seed(seed)
    c.pool.copy_(torch.randn(c.pool.shape, generator=g, device=dev))
    ids = torch.randperm(sum(need) + 3, generator=g, device=dev).int()
    for i, at in enumerate(np.concatenate([[0], np.cumsum(need)])[:-1].tolist()):
        c.table[i, :need[i]] = ids[at:at + need[i]]
    c.lens.copy_(_ints(lens, dev))
    c.refs[ids[:sum(need)].long()] = 1
    return c


def _check(got, q, c, seq, heads):
    """Rows of one sequence, (tokens, heads, dim), against the definition."""
    n, T, G = int(c.lens[seq]), q.shape[0], q.shape[1] // c.n_kv_heads
    pages = c.table[seq, :-(-n // c.page_size)].long()
    for h in heads:
        kv = c.pool[pages, 0, :, h // G].double().cpu().numpy()
        k, v = (kv[:, i].reshape(-1, c.head_dim)[:n] for i in (0, 1))
        s = k @ q[:, h].double().cpu().numpy().T * c.head_dim ** -0.5
        s[np.arange(n)[:, None] > n - T + np.arange(T)] = -np.inf
        w = np.exp(s - s.max(0))
        w /= w.sum(0)
        o, A = w.T @ v, w.T @ np.abs(v)
        err = np.abs(got[:, h].double().cpu().numpy() - o)
        assert (err <= 2.0 ** -8 * (A + np.abs(o)) + 2.0 ** -14 * A).all(), (seq, h, err.max())


def _q(dev, *shape):
    import torch
    return (2 * torch.randn(shape, generator=torch.Generator().manual_seed(9))).to(dev, torch.bfloat16)


@pytest.mark.parametrize("tokens,heads", [(1, 8), (3, 64), (9, 32)])     # 16, 32 and 128 rows to a tile
def test_runs_of_many_pages(gpu, tokens, heads):
    """8 heads of 150001 tokens over 512 blocks: 2300 keys, 146 pages of 16, to a run."""
    from tensorpack_amd.attention import cached_attention
    print("pages", tokens, heads, flush=True)
    c = _cache(gpu, [150001, 77], 8, 64)
    q = _q(gpu, 2, tokens, heads, 64)
    got = cached_attention(q, c, 0, _ints([0, 1], gpu))
    _check(got[0], q[0], c, 0, (0, heads // 2 + 1, heads - 1))
    _check(got[1], q[1], c, 1, range(heads))


@pytest.mark.parametrize("tokens,heads", [(3, 16), (5, 32)])             # 32 and 128 rows to a prefix tile
def test_prefixes_of_many_pages(gpu, tokens, heads):
    from tensorpack_amd.attention import cached_attention
    print("prefix pages", tokens, heads, flush=True)
    c = _cache(gpu, [150001, 10], 8, 64)
    c.table[1], c.lens[1] = c.table[0], 150001 - 20
    q = _q(gpu, 2, tokens, heads, 64)
    got = cached_attention(q, c, 0, _ints([0, 1], gpu), groups=_ints([0, 2], gpu), prefix_lens=_ints([149900], gpu))
    for s in (0, 1):
        _check(got[s], q[s], c, s, (0, heads - 1))


def test_single_waves_with_runs_of_many_pages(gpu):
    """4 heads of 120000 tokens beside 4100 short sequences: runs of single waves, 55 units of 32 keys each."""
    from tensorpack_amd.attention import cached_attention
    lens = [40 + i % 25 for i in range(4100)]
    lens[2000] = 120000
    c = _cache(gpu, lens, 4, 32)
    q = _q(gpu, len(lens), 1, 8, 32)
    got = cached_attention(q, c, 0, _ints(list(range(len(lens))), gpu))
    for s in (0, 1, 1999, 2000, 2001, 3000, 4099):
        _check(got[s], q[s], c, s, range(8))
    few = cached_attention(q[1990:2010], c, 0, _ints(list(range(1990, 2010)), gpu))
    for s in range(1990, 2010):
        _check(few[s - 1990], q[s], c, s, (0, 7))


@pytest.mark.parametrize("tokens,heads", [(1, 4), (5, 16)])
def test_more_sequences_than_the_lists_in_lds(gpu, tokens, heads):
    from tensorpack_amd.attention import cached_attention
    import torch
    print("sequences", tokens, heads, flush=True)
    members, common, n = 3, 32, 900
    c = _cache(gpu, [common + 1 + (37 * i) % 70 for i in range(n)], 2, 64)
    for i in range(n):
        if i % members:
            c.table[i, :2] = c.table[i - i % members, :2]
    q = _q(gpu, n, tokens, heads, 64)
    q_lens = [(i % (tokens + 1)) for i in range(n)]
    seqs = list(range(n))
    plain = cached_attention(q, c, 0, _ints(seqs, gpu), q_lens=_ints(q_lens, gpu))
    grouped = cached_attention(q, c, 0, _ints(seqs, gpu), q_lens=_ints(q_lens, gpu),
                               groups=_ints(list(range(0, n + 1, members)), gpu), prefix_lens=_ints([common] * (n // members), gpu))
    for got in (plain, grouped):
        assert torch.isfinite(got).all()
        for s in (0, 1, 2, 511, 512, 513, 700, 898, 899):
            k = q_lens[s]
            assert not got[s, k:].any()
            if k:
                _check(got[s, :k], q[s, :k], c, s, range(heads))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,K,V", [(33, 2, 128003), (3, 1, 1400003)])
def test_vocabularies_in_two_rounds(gpu, dtype, B, K, V):
    """B V of 2^22 and more. Random numbers have no ties within fp32's rounding: tokens are compared for equality."""
    import torch
    from tensorpack_amd.sampling import verify_drafts
    print("verify", dtype, B, K, V, flush=True)
    g = torch.Generator(device=gpu).manual_seed(V)
    dt = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    logits = torch.randn((B, K + 1, V), generator=g, device=gpu) * 2
    p = torch.softmax(logits, -1).to(dt)
    q32 = torch.softmax(logits[:, :K] + 0.5 * torch.randn((B, K, V), generator=g, device=gpu), -1)
    race = lambda *s: 1.0 / torch.empty(s, device=gpu).exponential_(generator=g).clamp_min(1e-20)
    drafts, q, noise = (q32 * race(B, K, V)).argmax(-1).int(), q32.to(dt), race(B, V)
    u = torch.rand((B, K), generator=g, device=gpu)
    tokens, accepted = (t.cpu().numpy() for t in verify_drafts(drafts, p, q, u, noise))
    d = drafts.cpu().numpy()
    counts = set()
    for b in range(B):
        n = 0
        while n < K and float(u[b, n]) * float(q[b, n, d[b, n]]) < float(p[b, n, d[b, n]]):
            n += 1
        w = p[b, n].double()
        if n < K:
            rest = (w - q[b, n].double()).clamp_min(0)
            w = rest if bool((rest > 0).any()) else w
        want = int((w * noise[b].double()).argmax())
        assert accepted[b] == n and tokens[b].tolist() == d[b, :n].tolist() + [want] + [-1] * (K - n)
        counts.add(n)
    assert len(counts) > 1 or B < 10
