"""PagedCache.reorder against lists: page ids, counts and lengths are compared for equality."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _ints(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _filled(dev, kind, lens, pages=300, width=40, seqs=None, seed=0):
    """A cache whose sequences hold `lens` tokens, each forked from the one before up to a random place."""
    import torch
    from tensorpack_amd.cache import PagedCache, QuantizedCache
    rng = np.random.RandomState(seed)
    seqs = seqs or len(lens)
    make = QuantizedCache if kind else PagedCache
    c = make(pages, 1, 1, 16, max_seqs=seqs, max_pages=width, page_size=16, device=dev)
    for i, n in enumerate(lens):
        if i and rng.rand() < 0.7:
            c.fork(_ints([i - 1], dev), _ints([i], dev))
            c.truncate(_ints([i], dev), _ints([min(n, rng.randint(0, lens[i - 1] + 1))], dev))
        c.extend(_ints([i], dev), _ints([n - int(c.lens[i])], dev))
    c.check()
    return c


def _state(c):
    return [c.table.cpu().numpy().copy(), c.lens.cpu().numpy().copy(), c.refs.cpu().numpy().copy()]


def _expect(state, seqs, parents, page=16):
    table, lens, refs = (x.copy() for x in state)
    rows = [(state[0][seqs[p]].copy(), state[1][seqs[p]]) for p in parents]
    for s, (row, n) in zip(seqs, rows):
        for p in state[0][s][:-(-state[1][s] // page)]:
            refs[p] -= 1
        for p in row[:-(-n // page)]:
            refs[p] += 1
        table[s], lens[s] = row, n
    return [table, lens, refs]


@pytest.mark.parametrize("kind", [False, True])
@pytest.mark.parametrize("n,width", [(1, 4), (4, 40), (7, 40), (40, 40), (300, 20), (1500, 8)])
def test_against_lists(gpu, kind, n, width):
    rng = np.random.RandomState(n)
    if n <= 40:
        lens = rng.randint(0, 16 * width + 1, n).tolist()
        lens[0] = 16 * width
        c = _filled(gpu, kind, lens, pages=n * width + 9, width=width, seqs=n + 5)
    else:
        import torch
        from tensorpack_amd.cache import PagedCache, QuantizedCache
        c = (QuantizedCache if kind else PagedCache)(n * width, 1, 1, 16, max_seqs=n + 5, max_pages=width, device=gpu)
        c.extend(_ints(list(range(n)), gpu), _ints(rng.randint(0, 16 * width + 1, n).tolist(), gpu))
    for trial in range(6):
        seqs = rng.permutation(n + 5)[:max(1, n - trial % 3)]
        m = len(seqs)
        parents = [np.arange(m), np.roll(np.arange(m), 1), rng.randint(0, m, m), np.zeros(m, int), rng.permutation(m), rng.randint(0, m, m)][trial]
        before = _state(c)
        c.reorder(_ints(seqs.tolist(), gpu), _ints(parents.tolist(), gpu))
        c.check()
        want = _expect(before, seqs, parents)
        got = _state(c)
        for a, b, what in zip(got, want, ("table", "lens", "refs")):
            assert np.array_equal(a, b), (what, trial)
        assert (got[2][:int(c.state[1])] > 0).all()              # no free page below the mark
    c.extend(_ints([0], gpu), _ints([0], gpu))
    c.check()


def test_long_tables(gpu):
    """More columns than the call's blocks take at a time (1200 sequences: one column a turn), far beyond most sequences."""
    import torch
    from tensorpack_amd.cache import PagedCache
    rng = np.random.RandomState(5)
    c = PagedCache(6000, 1, 1, 8, max_seqs=1200, max_pages=900, device=gpu)
    lens = rng.randint(0, 40, 1200)
    lens[[3, 700]] = 16 * 900, 16 * 600 + 1
    c.extend(_ints(list(range(1200)), gpu), _ints(lens.tolist(), gpu))
    c.check()
    for trial in range(3):
        seqs, parents = rng.permutation(1200), rng.randint(0, 1200, 1200)
        parents[:2] = [list(seqs).index(700), list(seqs).index(3)]
        before = _state(c)
        c.reorder(_ints(seqs.tolist(), gpu), _ints(parents.tolist(), gpu))
        c.check()
        assert all(np.array_equal(a, b) for a, b in zip(_state(c), _expect(before, seqs, parents)))


def test_then_extended(gpu):
    """Beams that take the same parent share its pages until they write."""
    import torch
    from tensorpack_amd.cache import PagedCache
    c = PagedCache(40, 1, 1, 16, max_seqs=4, max_pages=6, device=gpu)
    seqs = _ints([0, 1, 2, 3], gpu)
    c.extend(seqs, _ints([20, 21, 22, 23], gpu))
    cu = _ints([0, 20, 41, 63, 86], gpu)
    x = torch.randn((86, 1, 16), device=gpu).bfloat16()
    c.append(0, x, x, seqs, cu)
    held = [c.pool[c.table[s, :2].long(), 0, 0, 0].flatten(0, 1).clone() for s in range(4)]
    c.reorder(seqs, _ints([2, 2, 0, 2], gpu))
    c.extend(seqs, _ints([1, 1, 1, 1], gpu))
    y = torch.randn((4, 1, 16), device=gpu).bfloat16()
    c.append(0, y, y, seqs, _ints([0, 1, 2, 3, 4], gpu))
    c.check()
    for s, (p, n) in enumerate([(2, 22), (2, 22), (0, 20), (2, 22)]):
        now = c.pool[c.table[s, :2].long(), 0, 0, 0].flatten(0, 1)
        assert torch.equal(now[:n], held[p][:n]) and torch.equal(now[n], y[s, 0])
    assert c.lens.tolist() == [23, 23, 21, 23] and int((c.refs > 0).sum()) == 2 + 4       # two first pages, four last ones


def test_bad_lists_change_nothing(gpu):
    from tensorpack_amd.cache import CacheError
    c = _filled(gpu, False, [30, 40, 50], seqs=6)
    before = _state(c)
    for seqs, parents in (([0, 1, 0], [0, 0, 0]), ([0, 1, 6], [0, 0, 0]), ([0, -1], [0, 0]), ([0, 1], [0, 2]), ([0, 1], [-1, 0])):
        c.reorder(_ints(seqs, gpu), _ints(parents, gpu))
        with pytest.raises(CacheError) as e:
            c.check()
        assert e.value.bits == 1
        assert all(np.array_equal(a, b) for a, b in zip(_state(c), before))
    c.reorder(_ints([], gpu), _ints([], gpu))
    with pytest.raises(ValueError):
        c.reorder(_ints([0, 1], gpu), _ints([0], gpu))
    with pytest.raises(ValueError):
        c.reorder(_ints([0, 1], gpu), _ints([0, 1], gpu).long())


def test_capture(gpu):
    import torch
    c = _filled(gpu, True, [30, 0, 50, 64], seqs=5)
    seqs, parents = _ints([0, 1, 2, 3], gpu), _ints([0, 1, 2, 3], gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.reorder(seqs, parents)
    for p in ([1, 0, 3, 2], [0, 1, 2, 3], [2, 2, 2, 1], [0, 0, 1, 1]):
        parents.copy_(_ints(p, gpu))
        before = _state(c)
        graph.replay()
        assert all(np.array_equal(a, b) for a, b in zip(_state(c), _expect(before, [0, 1, 2, 3], p)))
        c.check()
