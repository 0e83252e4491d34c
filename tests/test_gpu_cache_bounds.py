"""Bookkeeping calls on a cache whose device arrays hold values that no call wrote. All arrays of the bookkeeping are
compared for equality (they lie one after another in one tensor, so that an index outside one shows in its neighbour)."""

import pytest

pytestmark = pytest.mark.gpu
TOP = (1 << 31) - 1


def _ints(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _fresh(dev, n_pages=40, max_seqs=6, max_pages=5):
    from tensorpack_amd.cache import PagedCache
    return PagedCache(n_pages, 1, 1, 64, max_seqs=max_seqs, max_pages=max_pages, device=dev)


def _refused(c, bits, call):
    import torch
    from tensorpack_amd.cache import CacheError
    before = c.book.clone()
    call()
    with pytest.raises(CacheError) as e:
        c.check()
    assert e.value.bits == bits
    assert torch.equal(c.book[4:], before[4:]) and c.state[1] == before[1]


@pytest.mark.parametrize("seq", [0, 3])
@pytest.mark.parametrize("length,count", [(-1, 1), (-40, 60), (-100, 200), (-TOP - 1, TOP)])
def test_extend_refuses_a_negative_length(gpu, seq, length, count):
    print("extend", seq, length, count, flush=True)
    c = _fresh(gpu)
    c.extend(_ints([1, 2], gpu), _ints([20, 3], gpu))
    c.lens[seq] = length
    _refused(c, 8, lambda: c.extend(_ints([seq], gpu), _ints([count], gpu)))
    _refused(c, 8, lambda: c.extend(_ints([1, seq], gpu), _ints([20, count], gpu)))


def test_lengths_above_the_table(gpu):
    c = _fresh(gpu)
    c.extend(_ints([0, 1], gpu), _ints([40, 70], gpu))
    c.lens[1] = TOP                                              # counts as 80: the five pages of its row
    _refused(c, 4, lambda: c.extend(_ints([1], gpu), _ints([1], gpu)))
    _refused(c, 8, lambda: c.truncate(_ints([1], gpu), _ints([TOP], gpu)))
    _refused(c, 8, lambda: c.truncate(_ints([1], gpu), _ints([81], gpu)))
    c.fork(_ints([1], gpu), _ints([4], gpu))
    assert c.table[4].tolist() == c.table[1].tolist() and c.lens[4] == 80
    assert c.refs.tolist() == [1] * 3 + [2] * 5 + [0] * 32
    c.free(_ints([1, 4], gpu))
    assert c.lens.tolist() == [40, 0, 0, 0, 0, 0] and c.refs.tolist() == [1] * 3 + [0] * 37
    assert c.table[1:].eq(-1).all()
    c.check()


def test_append_after_a_length_that_no_call_wrote(gpu):
    import torch
    c = _fresh(gpu)
    c.pool.zero_()
    c.extend(_ints([1], gpu), _ints([70], gpu))
    k = torch.ones((3, 1, 64), dtype=c.dtype, device=gpu)
    for length in (-TOP - 1, -5):
        c.lens[1] = length
        c.append(0, k, k, _ints([1], gpu), _ints([0, 3], gpu))
    assert not c.pool.any()
    c.lens[1] = TOP                                              # the last tokens of the row: 77, 78 and 79
    c.append(0, k, k, _ints([1], gpu), _ints([0, 3], gpu))
    page = int(c.table[1, 4])
    assert c.pool[page, 0, :, 0, 13:].eq(1).all() and c.pool.count_nonzero() == 2 * 3 * 64


@pytest.mark.parametrize("n_pages", [1, 3, 5, 63, 1000, 4095, 4096, 4097, 9001])
def test_compact_takes_the_pool_s_pages_only(gpu, n_pages):
    """Pools that the planning block's threads do not divide, after another pool's counts were in the same registers."""
    import torch
    from tensorpack_amd.cache import PagedCache
    print("compact", n_pages, flush=True)
    make = lambda n: PagedCache(n, 1, 1, 8, max_seqs=2, max_pages=n, device=gpu)
    full, c = make(8192), make(n_pages)
    full.refs.fill_(7)
    full.compact()
    pages = torch.randperm(n_pages, generator=torch.Generator().manual_seed(n_pages))[:(n_pages + 1) // 2].int().to(gpu)
    held = torch.arange(n_pages, device=gpu, dtype=c.dtype)[:, None, None, None, None, None].expand_as(c.pool)
    c.pool.copy_(held)
    c.table[1, :len(pages)], c.lens[1] = pages, 16 * len(pages)
    c.refs[pages.long()] = 1
    c.scratch.fill_(-5)
    want = pages.tolist()
    holes = [p for p in range(len(want)) if p not in set(want)]
    moved = dict(zip(sorted(p for p in want if p >= len(want)), holes))
    c.compact()
    assert c.table[1, :len(want)].tolist() == [moved.get(p, p) for p in want]
    assert c.refs.tolist() == [1] * len(want) + [0] * (n_pages - len(want))
    assert torch.equal(c.pool[c.table[1, :len(want)].long()], held[pages.long()])
    assert c.state.tolist() == [0, len(want), len(moved), 0]
    assert c.scratch[:len(moved)].tolist() == sorted(moved) and c.scratch[len(moved):n_pages].eq(-5).all()
    assert c.scratch[n_pages:n_pages + len(moved)].tolist() == holes and c.scratch[n_pages + len(moved):2 * n_pages].eq(-5).all()
    assert c.scratch[3 * n_pages:].eq(-5).all()
    c.check()


def test_compact_takes_negative_counts_as_free(gpu):
    import torch
    c = _fresh(gpu, n_pages=20)
    c.pool.copy_(torch.arange(20, device=gpu)[:, None, None, None, None, None].expand_as(c.pool))
    c.table[2, :4], c.lens[2] = _ints([19, 1, 7, 3], gpu), 60
    c.refs[c.table[2, :4].long()] = 1
    c.refs[0], c.refs[2], c.refs[5] = -1, -TOP - 1, -7
    c.scratch.fill_(TOP)
    c.compact()
    assert c.table[2].tolist() == [2, 1, 0, 3, -1] and c.refs[:4].tolist() == [1, 1, 1, 1]
    assert c.refs[4:].tolist() == [0, -7] + [0] * 14
    assert c.pool[:4, 0, 0, 0, 0, 0].tolist() == [7, 1, 19, 3]
    c.check()


def test_restore_leaves_the_status(gpu):
    import torch
    from tensorpack_amd.cache import CacheError
    c = _fresh(gpu)
    c.extend(_ints([0], gpu), _ints([20], gpu))
    clean = c.snapshot()
    c.extend(_ints([1, 1], gpu), _ints([1, 1], gpu))             # refused after the snapshot
    c.extend(_ints([2], gpu), _ints([30], gpu))
    c.restore(clean)
    assert c.lens.tolist() == [20, 0, 0, 0, 0, 0] and torch.equal(c.book[1:], clean[1:])
    pending = c.snapshot()                                       # with the refusal still to be reported
    with pytest.raises(CacheError) as e:
        c.check()
    assert e.value.bits == 1
    c.restore(pending)
    c.check()                                                    # reported once
