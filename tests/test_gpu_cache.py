"""PagedCache against the same bookkeeping written as plain lists. Everything is compared for equality: page ids,
counts, lengths and the pages' bits (append rounds fp32 input once, to nearest even, as torch does)."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _ints(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Model:
    """The cache's contract over lists: extend / fork / truncate / compact, pages as numpy arrays."""

    def __init__(self, cache):
        self.page, self.max_pages = cache.page_size, cache.max_pages
        self.rows = [[] for _ in range(cache.max_seqs)]
        self.lens = [0] * cache.max_seqs
        self.refs = [0] * cache.n_pages
        self.pool = self.bits(cache)

    @staticmethod
    def bits(cache):
        import torch
        return cache.pool.view(torch.int16).cpu().numpy().copy()

    def pages(self, n):
        return -(-n // self.page)

    def extend(self, seqs, counts):
        shared = [n % self.page > 0 and c > 0 and self.refs[self.rows[s][-1]] > 1
                  for s, c, n in ((s, c, self.lens[s]) for s, c in zip(seqs, counts))]
        free = [p for p, r in enumerate(self.refs) if r == 0]
        news = [self.pages(self.lens[s] + c) - self.pages(self.lens[s]) for s, c in zip(seqs, counts)]
        if any(self.pages(self.lens[s] + c) > self.max_pages for s, c in zip(seqs, counts)) or sum(news) + sum(shared) > len(free):
            return False
        free = iter(free)
        before = self.pool.copy()
        for s, c, copy, new in zip(seqs, counts, shared, news):
            if copy:
                p = next(free)
                self.refs[self.rows[s][-1]] -= 1
                self.pool[p] = before[self.rows[s][-1]]
                self.rows[s][-1], self.refs[p] = p, 1
            for _ in range(new):
                p = next(free)
                self.rows[s].append(p)
                self.refs[p] = 1
            self.lens[s] += c
        return True

    def fork(self, src, dst):
        for a, b in zip(src, dst):
            self.rows[b], self.lens[b] = list(self.rows[a]), self.lens[a]
            for p in self.rows[a]:
                self.refs[p] += 1

    def truncate(self, seqs, lens):
        for s, n in zip(seqs, lens):
            for p in self.rows[s][self.pages(n):]:
                self.refs[p] -= 1
            self.rows[s], self.lens[s] = self.rows[s][:self.pages(n)], n

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        move = dict(zip([p for p in range(live, len(self.refs)) if self.refs[p]], holes))
        for a, b in move.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.pool[b] = self.pool[a]
        self.rows = [[move.get(p, p) for p in r] for r in self.rows]

    def write(self, layer, k, v, seqs, cu):
        for i, s in enumerate(seqs):
            n = cu[i + 1] - cu[i]
            for j in range(n):
                at = self.lens[s] - n + j
                if at >= 0:
                    p = self.rows[s][at // self.page]
                    self.pool[p, layer, 0, :, at % self.page] = k[cu[i] + j]
                    self.pool[p, layer, 1, :, at % self.page] = v[cu[i] + j]

    def check(self, cache, what):
        table = np.full((len(self.rows), self.max_pages), -1)
        for i, r in enumerate(self.rows):
            table[i, :len(r)] = r
        assert np.array_equal(cache.lens.cpu().numpy(), self.lens), what
        assert np.array_equal(cache.refs.cpu().numpy(), self.refs), what
        assert np.array_equal(cache.table.cpu().numpy(), table), what
        assert np.array_equal(self.bits(cache), self.pool), what
        first = int(cache.state[1].item())
        assert all(self.refs[:first]), what                      # no free page below the mark


def _fresh(dev, n_pages=64, layers=2, kv=2, dim=64, page=16, max_seqs=24, max_pages=12, dtype=None, seed=0):
    import torch
    from tensorpack_amd.cache import PagedCache
    c = PagedCache(n_pages, layers, kv, dim, max_seqs=max_seqs, max_pages=max_pages, page_size=page, dtype=dtype, device=dev)
    g = torch.Generator().manual_seed(seed)
    c.pool.copy_(torch.randn(c.pool.shape, generator=g))
    return c, Model(c)


@pytest.mark.parametrize("page,dim,seed", [(16, 64, 0), (32, 40, 1), (64, 128, 2)])
def test_random_sequence_of_calls(gpu, page, dim, seed):
    import torch
    rng = np.random.RandomState(seed)
    c, m = _fresh(gpu, page=page, dim=dim, seed=seed, dtype=torch.float16 if seed == 1 else None)
    done = set()
    for step in range(120):
        held = [s for s in range(24) if m.lens[s]]
        empty = [s for s in range(24) if not m.lens[s]]
        op = rng.choice(["extend", "extend", "fork", "truncate", "free", "compact"])
        if op == "extend":
            seqs = rng.permutation(24)[:rng.randint(1, 9)].tolist()
            counts = [int(rng.choice([0, 1, 1, 2, page, page + 3, 3 * page])) for _ in seqs]
            before = c.book.clone()
            c.extend(_ints(seqs, gpu), _ints(counts, gpu))
            if not m.extend(seqs, counts):
                with pytest.raises(Exception) as e:
                    c.check()
                assert e.value.bits in (2, 4)
                assert torch.equal(c.book[4:], before[4:])       # nothing changed
                op = "refused"
        elif op == "fork" and held and empty:
            n = min(len(empty), rng.randint(1, 5))
            src, dst = rng.choice(held, n).tolist(), rng.permutation(empty)[:n].tolist()
            c.fork(_ints(src, gpu), _ints(dst, gpu))
            m.fork(src, dst)
        elif op == "truncate" and held:
            seqs = rng.permutation(held)[:3].tolist()
            lens = [int(rng.randint(0, m.lens[s] + 1)) for s in seqs]
            c.truncate(_ints(seqs, gpu), _ints(lens, gpu))
            m.truncate(seqs, lens)
        elif op == "free" and held:
            seqs = rng.permutation(held)[:2].tolist()
            c.free(_ints(seqs, gpu))
            m.truncate(seqs, [0] * len(seqs))
        elif op == "compact":
            c.compact()
            m.compact()
        m.check(c, (step, op))
        done.add(op)
    assert done >= {"extend", "fork", "truncate", "free", "compact"}
    c.check()


@pytest.mark.parametrize("src", ["fp32", "same", "views"])
@pytest.mark.parametrize("dim", [40, 128])
def test_append(gpu, src, dim):
    import torch
    c, m = _fresh(gpu, n_pages=200, dim=dim, max_pages=30, seed=4)
    seqs, counts = [3, 7, 1, 20, 9], [1, 0, 300, 16, 33]
    g = torch.Generator().manual_seed(8)
    for layer, part in ((1, None), (0, [1, 0, 5, 16, 2])):       # the whole prompt; the last tokens only
        if part is None:
            c.extend(_ints(seqs, gpu), _ints(counts, gpu))
            assert m.extend(seqs, counts)
        n = part or counts
        cu = np.concatenate([[0], np.cumsum(n)]).tolist()
        x = torch.randn((cu[-1], 4, dim), generator=g)
        x = x if src == "fp32" else x.to(c.dtype)
        x = x.to(gpu)
        k, v = x[:, :2], x[:, 2:]
        if src != "views":
            k, v = k.contiguous(), v.contiguous()
        c.append(layer, k, v, _ints(seqs, gpu), _ints(cu, gpu))
        bits = lambda t: t.to(c.dtype).view(torch.int16).cpu().numpy()
        m.write(layer, bits(k), bits(v), seqs, cu)
        m.check(c, layer)


def test_append_out_of_place_rows_write_nothing(gpu):
    import torch
    c, m = _fresh(gpu, seed=5)
    c.extend(_ints([2], gpu), _ints([5], gpu))
    assert m.extend([2], [5])
    k = torch.ones((9, 2, 64), dtype=c.dtype, device=gpu)
    m.write(0, np.full((9, 2, 64), k.view(torch.int16)[0, 0, 0].item()), np.full((9, 2, 64), k.view(torch.int16)[0, 0, 0].item()), [2], [0, 9])
    c.append(0, k, k, _ints([2], gpu), _ints([0, 9], gpu))       # four rows would fall before token 0
    m.check(c, "before token 0")
    c.append(0, k, k, _ints([5], gpu), _ints([0, 9], gpu))       # holds nothing
    c.append(0, k, k, _ints([-1, 99], gpu), _ints([0, 4, 9], gpu))
    c.append(0, k, k, _ints([2, 2], gpu), _ints([0, 0, 0], gpu))
    m.check(c, "nothing")


def test_large_lists(gpu):
    # more sequences than threads of the planning block, more pages than one of its rounds
    c, m = _fresh(gpu, n_pages=9000, layers=1, kv=1, dim=8, max_seqs=3000, max_pages=40, seed=6)
    rng = np.random.RandomState(0)
    seqs = rng.permutation(3000)[:2500].tolist()
    counts = rng.randint(0, 60, size=2500).tolist()
    counts[0], counts[2400] = 640, 639
    c.extend(_ints(seqs, gpu), _ints(counts, gpu))
    assert m.extend(seqs, counts)
    m.check(c, "extend")
    gone = seqs[::3]
    c.free(_ints(gone, gpu))
    m.truncate(gone, [0] * len(gone))
    src = [seqs[1]] * 400
    c.fork(_ints(src, gpu), _ints(gone[:400], gpu))
    m.fork(src, gone[:400])
    m.check(c, "fork")
    c.extend(_ints(gone[:400], gpu), _ints([1] * 400, gpu))
    assert m.extend(gone[:400], [1] * 400)
    m.check(c, "copies")
    c.compact()
    m.compact()
    m.check(c, "compact")


def test_copy_pages_and_snapshot(gpu):
    import torch
    a, ma = _fresh(gpu, n_pages=20, seed=1)
    b, mb = _fresh(gpu, n_pages=30, seed=2)
    a.copy_pages(_ints([29, 3, 99, -1, 5], gpu), _ints([0, 19, 1, 2, 77], gpu), source=b)   # the last three: out of range
    ma.pool[0], ma.pool[19] = mb.pool[29], mb.pool[3]
    ma.check(a, "from another cache")
    a.copy_pages(_ints([0, 0], gpu), _ints([4, 9], gpu))
    ma.pool[4] = ma.pool[9] = ma.pool[0]
    ma.check(a, "within")
    a.extend(_ints([0, 1], gpu), _ints([20, 40], gpu))
    snap = a.snapshot()
    was = a.table.clone(), a.lens.clone(), a.refs.clone()
    a.free(_ints([0], gpu))
    a.compact()
    a.restore(snap)
    assert all(torch.equal(x, y) for x, y in zip(was, (a.table, a.lens, a.refs)))


def test_refused_calls_change_nothing(gpu):
    import torch
    from tensorpack_amd.cache import CacheError
    c, m = _fresh(gpu, n_pages=10, max_pages=6)
    c.extend(_ints([0, 1], gpu), _ints([20, 40], gpu))           # 2 + 3 pages
    assert m.extend([0, 1], [20, 40])
    cases = [
        (1, lambda: c.extend(_ints([3, 3], gpu), _ints([1, 1], gpu))), (1, lambda: c.extend(_ints([24], gpu), _ints([1], gpu))),
        (1, lambda: c.truncate(_ints([0, -1], gpu), _ints([0, 0], gpu))), (1, lambda: c.free(_ints([1, 1], gpu))),
        (1, lambda: c.fork(_ints([0, 0], gpu), _ints([5, 5], gpu))), (1, lambda: c.fork(_ints([0, 77], gpu), _ints([5, 6], gpu))),
        (2, lambda: c.extend(_ints([2, 3], gpu), _ints([80, 16], gpu))),                   # 6 pages, 5 are free
        (4, lambda: c.extend(_ints([2, 3], gpu), _ints([1, 97], gpu))),
        (8, lambda: c.extend(_ints([2, 0], gpu), _ints([1, -1], gpu))), (8, lambda: c.truncate(_ints([0], gpu), _ints([21], gpu))),
        (8, lambda: c.truncate(_ints([1, 0], gpu), _ints([3, -1], gpu))),
        (16, lambda: c.fork(_ints([0], gpu), _ints([1], gpu))), (16, lambda: c.fork(_ints([2], gpu), _ints([2], gpu))),
        (16, lambda: c.fork(_ints([0, 4], gpu), _ints([4, 5], gpu))),
    ]
    for bits, call in cases:
        call()
        m.check(c, bits)
        with pytest.raises(CacheError) as e:
            c.check()
        assert e.value.bits == bits
        c.check()                                                # the status was taken
    assert c.free_pages == 5
    for bad in (lambda: c.extend(torch.tensor([0], device=gpu), _ints([1], gpu)), lambda: c.extend(_ints([0], gpu), _ints([1, 2], gpu)),
                lambda: c.append(2, *[torch.zeros(1, 2, 64, dtype=c.dtype, device=gpu)] * 2, _ints([0], gpu), _ints([0, 1], gpu)),
                lambda: c.append(0, *[torch.zeros(1, 2, 32, dtype=c.dtype, device=gpu)] * 2, _ints([0], gpu), _ints([0, 1], gpu)),
                lambda: c.append(0, *[torch.zeros(1, 2, 64, dtype=torch.float64, device=gpu)] * 2, _ints([0], gpu), _ints([0, 1], gpu)),
                lambda: c.append(0, *[torch.zeros(1, 2, 64, device=gpu)] * 2, _ints([0], gpu), _ints([0], gpu)),
                lambda: c.copy_pages(_ints([0], gpu), _ints([1], gpu), source=_fresh(gpu, dim=40)[0])):
        with pytest.raises(ValueError):
            bad()
    for kw in ({"page": 24}, {"dim": 12}, {"dim": 136}, {"max_seqs": 1 << 17}, {"n_pages": 0}, {"dtype": torch.float32}):
        with pytest.raises(ValueError):
            _fresh(gpu, **kw)


def test_a_step_in_a_graph(gpu):
    # fork, extend, append and free recorded once and replayed, with other calls between
    import torch
    c, m = _fresh(gpu, n_pages=40, seed=9)
    c.extend(_ints([0], gpu), _ints([21], gpu))
    m.extend([0], [21])
    src, dst, one, cu = _ints([0, 0], gpu), _ints([1, 2], gpu), _ints([1, 1], gpu), _ints([0, 1, 2], gpu)
    k = torch.randn((2, 2, 64), device=gpu)
    bits = k.to(c.dtype).view(torch.int16).cpu().numpy()

    def step():
        c.free(dst)
        c.fork(src, dst)
        c.extend(dst, one)
        c.append(1, k, k, dst, cu)

    def plain():
        m.truncate([1, 2], [0, 0])
        m.fork([0, 0], [1, 2])
        assert m.extend([1, 2], [1, 1])
        m.write(1, bits, bits, [1, 2], [0, 1, 2])

    step()
    plain()
    m.check(c, "eager")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(4):
        g.replay()
        plain()
        m.check(c, i)
        c.extend(_ints([0], gpu), _ints([7], gpu))
        m.extend([0], [7])
    c.check()
