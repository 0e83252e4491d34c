"""QuantizedCache against its definition in numpy. Everything is compared for equality: exponents, codes, values read back, and what
a call must leave alone. (Steps are powers of two, so a value divided by one is exact in fp32 and its rounding is the same in any
precision.)"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

RANGE = {"bfloat16": (-100, 100), "float16": (-24, 9)}


def _ints(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _exponent(x, dtype):
    """Least e with max |x| <= 127 * 2 ** e over the finite values of x, in the type's range."""
    lo, hi = RANGE[dtype]
    x = np.abs(x[np.isfinite(x)])
    top = float(x.max()) if x.size else 0.0
    e = lo
    while e < hi and top > 127.0 * 2.0 ** e:
        e += 1
    return e


def _codes(x, e):
    with np.errstate(invalid="ignore"):
        return np.nan_to_num(np.clip(np.rint(x.astype(np.float64) * 2.0 ** -e), -127, 127), nan=0.0).astype(np.int64)


class Model:
    """Tokens of each sequence, as (codes, exponents) by block: [layer][K, V][head]."""

    def __init__(self, layers, kv, dim, dtype):
        self.shape, self.dtype = (layers, 2, kv), dtype
        self.dim, self.seqs = dim, {}

    def extend(self, s, n):
        codes, exps = self.seqs.setdefault(s, (np.zeros(self.shape + (0, self.dim), np.int64), np.zeros(self.shape + (0,), np.int64)))
        blocks = -(-(codes.shape[3] + n) // 16) - exps.shape[3]
        self.seqs[s] = (np.concatenate([codes, np.zeros(self.shape + (n, self.dim), np.int64)], 3),
                        np.concatenate([exps, np.zeros(self.shape + (blocks,), np.int64)], 3))

    def truncate(self, s, n):
        codes, exps = self.seqs[s]
        self.seqs[s] = codes[:, :, :, :n].copy(), exps[:, :, :, :-(-n // 16)].copy()

    def fork(self, a, b):
        self.seqs[b] = tuple(x.copy() for x in self.seqs[a])

    def append(self, layer, s, kv):
        """kv (2, n, heads, dim): the last n tokens."""
        codes, exps = self.seqs[s]
        n, m = kv.shape[1], codes.shape[3]
        kv, first = kv[:, max(n - m, 0):], max(m - n, 0)
        for b in range(first // 16, -(-m // 16)):
            at = max(first, 16 * b)
            old = at - 16 * b
            new = kv[:, at - first:min(m, 16 * b + 16) - first]
            for j in (0, 1):
                for h in range(self.shape[2]):
                    e = _exponent(new[j][:, h], self.dtype)
                    if old:
                        was = int(exps[layer, j, h, b])
                        e = max(e, was)
                        codes[layer, j, h, 16 * b:at] = _codes(codes[layer, j, h, 16 * b:at], e - was)
                    exps[layer, j, h, b] = e
                    codes[layer, j, h, at:at + new.shape[1]] = _codes(new[j][:, h], e)

    def values(self, layer, s, j):
        """(tokens, heads, dim)"""
        codes, exps = self.seqs[s]
        steps = 2.0 ** exps[layer, j].repeat(16, -1)[:, :codes.shape[3]]
        return (codes[layer, j] * steps[..., None]).transpose(1, 0, 2)

    def check(self, cache, what):
        import torch
        table, codes = cache.table.cpu().numpy(), cache.codes.cpu().numpy()
        scales = cache.scales.float().cpu().numpy()
        for s, (want, exps) in self.seqs.items():
            n = want.shape[3]
            assert int(cache.lens[s]) == n, what
            for i in range(n):
                p, at = table[s, i // cache.page_size], i % cache.page_size
                assert np.array_equal(codes[p, :, :, :, at], want[:, :, :, i]), (what, s, i)
                assert np.array_equal(scales[p, :, :, :, at // 16], 2.0 ** exps[:, :, :, i // 16]), (what, s, i)


def _cache(dev, dtype="bfloat16", pages=64, layers=2, kv=2, dim=64, page=16, seqs=12, width=12, fill=True):
    import torch
    from tensorpack_amd.cache import QuantizedCache
    c = QuantizedCache(pages, layers, kv, dim, max_seqs=seqs, max_pages=width, page_size=page, dtype=getattr(torch, dtype), device=dev)
    if fill:                                                     # whatever memory holds
        c.pool.copy_(torch.randint(-128, 128, c.pool.shape, generator=torch.Generator().manual_seed(1), dtype=torch.int8))
    return c, Model(layers, kv, dim, dtype)


def _rows(rng, n, kv, dim, spread=2.0):
    """Tokens of very different sizes, some of them zero."""
    x = rng.randn(2, n, kv, dim) * np.exp(spread * rng.randn(2, n, kv, 1)) * (rng.rand(2, n, kv, 1) > 0.1)
    return x.astype(np.float32)


def _upload(x, dtype, dev):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).to(getattr(torch, dtype))
    return t.to(dev), t.double().numpy()


@pytest.mark.parametrize("dtype,src,page,kv,dim", [("bfloat16", "bfloat16", 16, 2, 64), ("bfloat16", "float32", 32, 1, 40), ("float16", "float16", 64, 3, 128),
                                                   ("float16", "float32", 16, 5, 24), ("bfloat16", "bfloat16", 128, 1, 8), ("float16", "float16", 16, 2, 112)])
def test_random_calls(gpu, dtype, src, page, kv, dim):
    rng = np.random.RandomState(page + dim)
    c, m = _cache(gpu, dtype, kv=kv, dim=dim, page=page, pages=200)
    for step in range(40):
        live = [s for s in range(12) if s in m.seqs and m.seqs[s][0].shape[3]]
        op = rng.choice(["write"] * 5 + ["fork", "truncate", "compact", "free"])
        if op == "write":
            seqs = rng.permutation(12)[:rng.randint(1, 6)].tolist()
            counts = [int(rng.choice([0, 1, 1, 2, 15, 16, 17, 37])) for _ in seqs]
            counts = [n if (m.seqs[s][0].shape[3] if s in m.seqs else 0) + n <= 12 * page else 0 for s, n in zip(seqs, counts)]
            cu = np.concatenate([[0], np.cumsum(counts)]).tolist()
            c.extend(_ints(seqs, gpu), _ints(counts, gpu))
            for s, n in zip(seqs, counts):
                m.extend(s, n)
            for layer in (0, 1):
                (k, kd), (v, vd) = (_upload(x, src, gpu) for x in _rows(rng, cu[-1], kv, dim))
                for again in range(rng.randint(1, 3)):           # the same tokens again: nothing changes
                    c.append(layer, k, v, _ints(seqs, gpu), _ints(cu, gpu))
                for i, s in enumerate(seqs):
                    m.append(layer, s, np.stack([kd[cu[i]:cu[i + 1]], vd[cu[i]:cu[i + 1]]]))
        elif op == "fork" and live and len(live) < 12:
            a, b = rng.choice(live), rng.choice([s for s in range(12) if s not in live])
            c.fork(_ints([a], gpu), _ints([b], gpu))
            m.fork(a, b)
        elif op == "truncate" and live:
            s = int(rng.choice(live))
            n = rng.randint(0, m.seqs[s][0].shape[3] + 1)
            c.truncate(_ints([s], gpu), _ints([n], gpu))
            m.truncate(s, n)
        elif op == "free" and live:
            s = int(rng.choice(live))
            c.free(_ints([s], gpu))
            m.truncate(s, 0)
        elif op == "compact":
            c.compact()
        c.check()
        if step % 8 == 7 or step == 39:
            m.check(c, (step, op))
    seqs = [s for s in range(12) if s in m.seqs]
    lens = [m.seqs[s][0].shape[3] for s in seqs]
    cu = _ints(np.concatenate([[0], np.cumsum(lens)]).tolist(), gpu)
    import torch
    for layer in (0, 1):
        for out in (None, torch.float32):
            for j, x in enumerate(c.read(layer, _ints(seqs, gpu), cu, sum(lens), dtype=out)):
                want = np.concatenate([m.values(layer, s, j) for s in seqs])
                assert x.dtype == (out or getattr(torch, dtype)) and np.array_equal(x.double().cpu().numpy(), want)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_edges_of_the_scales(gpu, dtype):
    """A block for each largest value: 0, the smallest and largest of the type, 127 times powers of two and the next numbers
    beyond, ties of the rounding, infinities and NaN."""
    import torch
    t = getattr(torch, dtype)
    big = torch.finfo(t).max
    tops = [0.0, 127 * 2.0 ** -20, 127 * 2.0 ** -20 * (1 + torch.finfo(t).eps), 127.0, 127.5 if dtype == "float16" else 128.0, 254.0, 1.0, 2.0 ** -24, 3 * 2.0 ** -24,
            float(torch.finfo(t).tiny), big, -big, 65024.0, 65280.0, 60000.0, 1e-30 if dtype == "bfloat16" else 6e-8, 1e33 if dtype == "bfloat16" else 3e4]
    x = np.zeros((2, 16 * len(tops) + 32, 1, 64), np.float32)
    for i, top in enumerate(tops):
        x[:, 16 * i:16 * i + 16, 0] = np.linspace(-1, 1, 16 * 64).reshape(16, 64).astype(np.float32) * min(abs(top), 3e38)
        x[:, 16 * i + 3, 0, 5] = top
        e = _exponent(np.array([top]), dtype)
        x[:, 16 * i + 4, 0, :8] = np.array([0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -125.5, 0.0]) * 2.0 ** min(e, 7)
    a, b = 16 * len(tops), 16 * len(tops) + 16
    x[:, a:] = np.random.RandomState(0).randn(2, 32, 1, 64)
    x[:, a, 0, :3] = [math.nan, math.inf, -math.inf]
    x[:, b:] = math.nan
    x[:, b, 0, 0] = math.inf
    c, m = _cache(gpu, dtype, kv=1, layers=1, pages=40, width=32)
    (k, kd), (v, vd) = (_upload(y, dtype, gpu) for y in x)
    n = x.shape[1]
    c.extend(_ints([0], gpu), _ints([n], gpu))
    c.append(0, k, v, _ints([0], gpu), _ints([0, n], gpu))
    m.extend(0, n)
    m.append(0, 0, np.stack([kd, vd]))
    m.check(c, dtype)
    got = c.read(0, _ints([0], gpu), _ints([0, n], gpu), n)[0]
    assert torch.isfinite(got).all() and np.array_equal(got.double().cpu().numpy(), m.values(0, 0, 0))
    assert (got[a, 0, :3].cpu().double() == torch.tensor([0.0, 127.0, -127.0]) * 2.0 ** int(m.seqs[0][1][0, 0, 0, a // 16])).all()
    # one token after another: codes rounded again as larger ones come, steps from one end of the range to the other
    order = np.argsort([abs(t) for t in tops])
    y = x[:, [16 * i + 3 for i in order]][:, :16]
    (k, kd), (v, vd) = (_upload(z, dtype, gpu) for z in y)
    for i in range(16):
        c.extend(_ints([1], gpu), _ints([1], gpu))
        c.append(0, k[i:i + 1], v[i:i + 1], _ints([1], gpu), _ints([0, 1], gpu))
        m.extend(1, 1)
        m.append(0, 1, np.stack([kd[i:i + 1], vd[i:i + 1]]))
    m.check(c, "grown")
    c.check()


def test_error_is_half_a_step(gpu):
    """Values that are written once are off by half a step, at most 1 / 127 of their block's largest."""
    import torch
    rng = np.random.RandomState(5)
    c, _ = _cache(gpu, "bfloat16", layers=1, kv=4, dim=128, page=64, pages=20)
    x = torch.from_numpy(rng.randn(300, 4, 128).astype(np.float32)).to(gpu)
    c.extend(_ints([3], gpu), _ints([300], gpu))
    c.append(0, x, x, _ints([3], gpu), _ints([0, 300], gpu))
    got = c.read(0, _ints([3], gpu), _ints([0, 300], gpu), 300, dtype=torch.float32)[1]
    for b in range(0, 300, 16):
        y = x[b:b + 16]
        top = y.abs().amax((0, 2))
        assert ((got[b:b + 16] - y).abs().amax((0, 2)) <= top / 127).all()


def test_read_windows(gpu):
    """The last tokens of sequences in any order, more rows than tokens, rows of no sequence, strided results."""
    import torch
    rng = np.random.RandomState(7)
    c, m = _cache(gpu, "float16", kv=2, dim=40, page=32)
    lens = [70, 0, 5, 33]
    c.extend(_ints([0, 1, 2, 3], gpu), _ints(lens, gpu))
    cu = [0, 70, 70, 75, 108]
    (k, kd), (v, vd) = (_upload(x, "float16", gpu) for x in _rows(rng, 108, 2, 40, 0.5))
    c.append(1, k, v, _ints([0, 1, 2, 3], gpu), _ints(cu, gpu))
    for s in range(4):
        m.extend(s, lens[s])
        m.append(1, s, np.stack([kd[cu[s]:cu[s + 1]], vd[cu[s]:cu[s + 1]]]))
    back = [3, 3, 20, 20, 21, 60]                                # rows 0:3 and 60: belong to nobody; sequence 2 has 5 tokens, asked 17
    order = [0, 2, 1, 3, 0]
    for stride in (80, 96):
        buf = torch.full((2, 64, stride), 7.0, dtype=torch.float16, device=gpu)
        out = tuple(b[:, :80].unflatten(1, (2, 40)) for b in buf)
        got = c.read(1, _ints(order, gpu), _ints(back, gpu), out=out)
        assert got[0] is out[0]
        for j in (0, 1):
            want = np.full((64, 2, 40), 7.0)
            for i, s in enumerate(order):
                n = back[i + 1] - back[i]
                have = min(n, lens[s])
                want[back[i]:back[i + 1] - have] = 0
                want[back[i + 1] - have:back[i + 1]] = m.values(1, s, j)[lens[s] - have:]
            assert np.array_equal(out[j].double().cpu().numpy(), want)
        assert (buf[:, :, 80:] == 7.0).all()
    assert c.read(0, _ints([], gpu), _ints([0], gpu), 0)[0].shape == (0, 2, 40)
    bad = c.read(1, _ints([-1, 99], gpu), _ints([0, 2, 4], gpu), 4)
    assert not bad[0].any() and not bad[1].any()
    far = torch.full((2, 8, 2, 40), 3.0, dtype=torch.float16, device=gpu)
    c.read(1, _ints([0, 3], gpu), _ints([-5, 4, 1 << 30], gpu), out=tuple(far))          # offsets are cut at the rows
    assert np.array_equal(far[0].double().cpu().numpy(), np.concatenate([m.values(1, 0, 0)[-4:], m.values(1, 3, 0)[-4:]]))


def test_rows_far_apart(gpu):
    """K and V, and results, of rows 2 GiB apart: offsets pass 32 bits."""
    import torch
    c, _ = _cache(gpu, kv=2, dim=40)
    buf = torch.empty((3 << 30) + 4096, dtype=torch.bfloat16, device=gpu)
    far = lambda at: buf.as_strided((4, 2, 40), (1 << 30, 40, 1), at)
    near = torch.randn((2, 4, 2, 40), generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    k, v, to = far(0), far(256), (far(512), far(768))
    k.copy_(near[0])
    v.copy_(near[1])
    seqs, cu = _ints([0, 1], gpu), _ints([0, 3, 4], gpu)
    c.extend(seqs, _ints([3, 1], gpu))
    c.append(0, k, v, seqs, cu)
    c.append(1, near[0], near[1], seqs, cu)
    c.check()
    want = c.read(1, seqs, cu, 4)
    c.read(0, seqs, cu, out=to)
    assert all(torch.equal(a, b) for a, b in zip(to, want)) and all(bool(x.any(-1).all()) for x in want)


def test_more_rows_than_tokens(gpu):
    """Rows that would fall before token 0 are left out, and have no part in the scales."""
    rng = np.random.RandomState(8)
    c, m = _cache(gpu)
    c.extend(_ints([4], gpu), _ints([20], gpu))
    m.extend(4, 20)
    x = _rows(rng, 30, 2, 64, 0.3)
    x[:, :10] *= 1000
    (k, kd), (v, vd) = (_upload(y, "bfloat16", gpu) for y in x)
    for layer in (0, 1):
        c.append(layer, k, v, _ints([4], gpu), _ints([0, 30], gpu))
        m.append(layer, 4, np.stack([kd, vd]))
    m.check(c, "30 rows for 20 tokens")


def test_what_append_refuses(gpu):
    """Pages of several holders and sequences named twice get nothing; the call's other sequences do."""
    import torch
    from tensorpack_amd.cache import CacheError
    rng = np.random.RandomState(9)
    c, m = _cache(gpu)
    lens = [20, 20, 20]
    c.extend(_ints([0, 1, 2], gpu), _ints(lens, gpu))
    c.fork(_ints([0], gpu), _ints([5], gpu))
    (k, kd), (v, vd) = (_upload(x, "bfloat16", gpu) for x in _rows(rng, 60, 2, 64))
    before = c.pool.clone()
    c.append(0, k, v, _ints([0, 1, 2], gpu), _ints([0, 20, 40, 60], gpu))
    with pytest.raises(CacheError) as e:
        c.check()
    assert e.value.bits == 32
    rows = c.table[0, :2].long()
    assert torch.equal(c.pool[rows], before[rows])
    before = c.pool.clone()
    c.append(0, k, v, _ints([1, 2, 1], gpu), _ints([0, 20, 40, 60], gpu))
    with pytest.raises(CacheError) as e:
        c.check()
    assert e.value.bits == 1
    rows = c.table[1, :2].long()
    assert torch.equal(c.pool[rows], before[rows])
    got = c.read(0, _ints([2], gpu), _ints([0, 20], gpu), 20)[0]
    m.extend(2, 20)
    m.append(0, 2, np.stack([kd[20:40], vd[20:40]]))
    assert np.array_equal(got.double().cpu().numpy(), m.values(0, 2, 0))
    c.append(0, k, v, _ints([2, -1, 50], gpu), _ints([0, 20, 40, 60], gpu))          # out of range: nobody's rows
    c.append(0, k[:0], v[:0], _ints([2], gpu), _ints([0, 0], gpu))
    c.append(0, k, v, _ints([1, 2, 1], gpu), _ints([0, 20, 40, 40], gpu))            # the second time without rows
    c.check()


def test_copies_between_caches_and_snapshots(gpu):
    import torch
    from tensorpack_amd.cache import PagedCache, QuantizedCache
    rng = np.random.RandomState(10)
    c, m = _cache(gpu, kv=1, dim=40, page=16)
    d, _ = _cache(gpu, kv=1, dim=40, page=16, pages=9)
    d.copy_pages(_ints([3, 60, 99], gpu), _ints([8, 0, 1], gpu), c)
    assert torch.equal(d.pool[8], c.pool[3]) and torch.equal(d.pool[0], c.pool[60])
    for other in (PagedCache(4, 2, 1, 40, max_seqs=2, max_pages=2, device=gpu), _cache(gpu, kv=1, dim=48, page=16, pages=9)[0],
                  _cache(gpu, "float16", kv=1, dim=40, page=16, pages=9)[0]):
        with pytest.raises(ValueError):
            c.copy_pages(_ints([0], gpu), _ints([0], gpu), other)
    c.extend(_ints([0], gpu), _ints([50], gpu))
    (k, kd), (v, vd) = (_upload(x, "bfloat16", gpu) for x in _rows(rng, 50, 1, 40))
    for layer in (0, 1):
        c.append(layer, k, v, _ints([0], gpu), _ints([0, 50], gpu))
    e = QuantizedCache.from_buffers(c.pool, c.table, c.lens, c.refs, n_layers=2, n_kv_heads=1, head_dim=40, page_size=16)
    s = e.snapshot()
    a = e.read(1, _ints([0], gpu), _ints([0, 50], gpu), 50)
    e.free(_ints([0], gpu))
    e.restore(s)
    b = e.read(1, _ints([0], gpu), _ints([0, 50], gpu), 50)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and e.free_pages == c.free_pages


def test_views_and_capture(gpu):
    """K and V as views of one product's result, and a captured step (room, append, read) replayed on new tokens."""
    import torch
    rng = np.random.RandomState(11)
    c, m = _cache(gpu, layers=1)
    qkv = torch.from_numpy(rng.randn(3, (4 + 2 + 2) * 64).astype(np.float32)).bfloat16().to(gpu)
    k, v = (qkv[:, a:a + 128].unflatten(1, (2, 64)) for a in (256, 384))
    seqs, one, cu = _ints([2, 0, 7], gpu), _ints([1, 1, 1], gpu), _ints([0, 1, 2, 3], gpu)
    out = tuple(torch.empty((3, 2, 64), dtype=torch.bfloat16, device=gpu) for _ in (0, 1))

    def step():
        c.extend(seqs, one)
        c.append(0, k, v, seqs, cu)
        c.read(0, seqs, cu, out=out)

    def follow():
        for i, s in enumerate([2, 0, 7]):
            m.extend(s, 1)
            m.append(0, s, np.stack([x[i:i + 1].double().cpu().numpy() for x in (k, v)]))
            assert np.array_equal(out[0][i].double().cpu().numpy(), m.values(0, s, 0)[-1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    follow()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(20):
        qkv.copy_(torch.from_numpy(rng.randn(*qkv.shape).astype(np.float32) * 2.0 ** (i % 5)))
        graph.replay()
        follow()
        c.check()
    m.check(c, "replayed")
    odd = torch.randn((3, 64, 2), device=gpu).bfloat16().transpose(1, 2)             # copied first
    c.append(0, odd, odd, seqs, cu)
    d, n = _cache(gpu, layers=1)
    d.extend(seqs, one)
    d.append(0, odd.contiguous(), odd.contiguous(), seqs, cu)
    e, _ = _cache(gpu, layers=1)
    e.extend(seqs, one)
    e.append(0, odd, odd, seqs, cu)
    assert all(torch.equal(a, b) for a, b in zip(d.read(0, seqs, cu, 3), e.read(0, seqs, cu, 3)))


def test_many_short_and_long(gpu):
    """Batches whose blocks are numbered over the whole list: 1500 sequences of 0 to 40 new tokens, and one of 5000."""
    import torch
    rng = np.random.RandomState(12)
    c, m = _cache(gpu, pages=6000, layers=1, kv=1, dim=16, seqs=1501, width=320, fill=False)
    counts = rng.randint(0, 41, 1501)
    counts[700], counts[1500] = 5000, 17
    cu = np.concatenate([[0], np.cumsum(counts)])
    seqs = rng.permutation(1501)
    c.extend(_ints(seqs.tolist(), gpu), _ints(counts.tolist(), gpu))
    (k, kd), (v, vd) = (_upload(x, "bfloat16", gpu) for x in _rows(rng, int(cu[-1]), 1, 16))
    c.append(0, k, v, _ints(seqs.tolist(), gpu), _ints(cu.tolist(), gpu))
    c.check()
    got = [x.double().cpu().numpy() for x in c.read(0, _ints(seqs.tolist(), gpu), _ints(cu.tolist(), gpu), int(cu[-1]))]
    for i in list(range(0, 1501, 37)) + [700, 1500]:
        m.extend(i, int(counts[i]))
        m.append(0, i, np.stack([kd[cu[i]:cu[i + 1]], vd[cu[i]:cu[i + 1]]]))
        for j in (0, 1):
            assert np.array_equal(got[j][cu[i]:cu[i + 1]], m.values(0, i, j)), i


def test_refusals(gpu):
    import torch
    from tensorpack_amd.cache import QuantizedCache
    c, _ = _cache(gpu)
    s, cu, k = _ints([0], gpu), _ints([0, 4], gpu), torch.zeros((4, 2, 64), dtype=torch.bfloat16, device=gpu)
    for bad in (dict(layer=2), dict(layer=-1), dict(k=k.half(), v=k.half()), dict(k=k[:, :1]), dict(v=k[:3]), dict(k=k[..., :32], v=k[..., :32]),
                dict(seqs=s.long()), dict(cu=cu[:1]), dict(k=k.cpu(), v=k.cpu())):
        kw = {**dict(layer=0, k=k, v=k, seqs=s, cu=cu), **bad}
        with pytest.raises(ValueError):
            c.append(**kw)
    for bad in (dict(layer=2), dict(rows=-1), dict(rows=None), dict(dtype=torch.float16), dict(out=(k, k), rows=4), dict(rows=None, out=(k, k[:3])),
                dict(rows=None, out=(k, k[:1].expand(4, 2, 64))), dict(rows=None, out=(k.float(), k)), dict(rows=None, out=(k.half(), k.half())),
                dict(cu=cu.long()), dict(seqs=_ints([0, 1], gpu))):
        kw = {**dict(layer=0, seqs=s, cu=cu, rows=4), **bad}
        with pytest.raises(ValueError):
            c.read(**kw)
    for bad in (dict(head_dim=60), dict(head_dim=136), dict(page_size=8), dict(dtype=torch.float32), dict(n_pages=0)):
        kw = {**dict(n_pages=4, n_layers=1, n_kv_heads=1, head_dim=64, max_seqs=2, max_pages=2, device=gpu), **bad}
        with pytest.raises(ValueError):
            QuantizedCache(**kw)
    with pytest.raises(ValueError):
        QuantizedCache(4, 1, 1, 64, max_seqs=2, max_pages=2, pool=torch.zeros((4, 100), dtype=torch.int8, device=gpu))
