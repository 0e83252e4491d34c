"""Results that share memory with each other, or with what a call still reads, are refused, without a GPU: apply_rotary's and
QuantizedCache.read's checks, and the question that both ask, against a count of every element's address."""

import itertools

import numpy as np
import pytest
import torch

from tensorpack_amd import attention, rotary


def _handle(x):
    return x.data_ptr(), x.stride(0), x.stride(1)


def _elements(x):
    at = torch.arange(x.untyped_storage().nbytes() // x.element_size()).as_strided(x.shape, x.stride(), x.storage_offset())
    return set(at.flatten().tolist())


def _views():
    x = torch.zeros(6000, dtype=torch.bfloat16)
    for rows, heads, dim, r, h, at in itertools.product((1, 2, 5), (1, 3), (8,), (8, 24, 48, 0, 1000), (8, 16, 40, 120), (0, 8, 24, 48, 1000)):
        yield x.as_strided((rows, heads, dim), (r, h, 1), at)


def test_whether_views_meet():
    views = list(_views())
    held = [_elements(v) for v in views]
    rng = np.random.RandomState(0)
    found = [0, 0]
    for i, j in rng.randint(0, len(views), (6000, 2)):
        a, b = views[i], views[j]
        want = bool(held[i] & held[j])
        assert attention._meet(_handle(a), a.shape, _handle(b), b.shape, 2) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        found[want] += 1
    assert min(found) > 500
    none = torch.zeros((0, 2, 8), dtype=torch.bfloat16)
    assert not attention._meet(_handle(none), none.shape, _handle(views[0]), views[0].shape, 2)


class _Cpu:
    device, dim, interleaved, amplitude, turns_at = torch.device("cpu"), 64, False, 1.0, 0


def test_rotary_results():
    x = torch.zeros((5, 8 * 64))
    q, k = (t.unflatten(1, (-1, 64)) for t in x.split([256, 256], dim=1))
    square = torch.zeros((4, 4, 64))
    long = torch.zeros((6, 4, 64))
    positions = torch.zeros(6, dtype=torch.int32)
    for q_, k_, out in ((square, None, (square.transpose(0, 1), None)), (long[:4], None, (long[1:5], None)), (long[1:5], None, (long[:4], None)),
                        (q, k, (k, q)), (q, k, (q, q)), (q, k, (torch.empty_like(q), q)), (q, k, (k, torch.empty_like(q))), (q, q, (q, q)),
                        (long[:4], long[2:], (torch.empty((4, 4, 64)), long[:4])), (torch.empty((4, 4, 64)), long[:4], (long[2:], torch.empty((4, 4, 64)))),
                        (square, torch.empty((4, 4, 64)), (long[:4], long[2:])),
                        (square[:, :2], None, (square[:, 1:3], None)), (square[:, :, :64], None, (square.flatten()[64:832].view(4, 3, 64)[:, :2], None))):
        with pytest.raises(ValueError):
            rotary.apply_rotary(_Cpu, q_, k_, positions[:q_.shape[0]], out=out)
    y = torch.zeros((5, 16 * 64))
    parts = [t.unflatten(1, (-1, 64)) for t in y.split([256] * 4, dim=1)]
    clash = lambda q, oq, k, ok: rotary._clash(_handle(q), _handle(oq), q.shape[1], _handle(k), _handle(ok), k.shape[1], q.shape[0], 64, 4)
    assert not clash(q, q, k, k) and not clash(q, parts[0], k, parts[1]) and not clash(q, q, k, parts[2]) and not clash(parts[3], parts[0], parts[2], parts[1])
    one = torch.zeros((1, 4, 64))                                   # a stride of an axis of one element says nothing
    assert not clash(one, one.as_strided((1, 4, 64), (64, 64, 1)), torch.zeros((1, 2, 64)), torch.zeros((1, 2, 64)))
    heads_first = torch.zeros((6, 5, 64)).transpose(0, 1)
    assert not clash(heads_first[:, :4], heads_first[:, :4], heads_first[:, 4:], heads_first[:, 4:])


def test_read_results():
    from tensorpack_amd.cache import QuantizedCache
    cache = object.__new__(QuantizedCache)
    cache.n_layers, cache.n_kv_heads, cache.head_dim, cache.dtype, cache.device = 1, 2, 64, torch.bfloat16, torch.device("cpu")
    seqs, cu = torch.zeros(1, dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    x = torch.zeros((8, 2, 64), dtype=torch.bfloat16)
    for k, v in ((x[:5], x[:5]), (x[:5], x[3:]), (x[3:], x[:5]), (x[:5].float(), x[:5].float()[:4])):
        with pytest.raises(ValueError):
            cache.read(0, seqs, cu, out=(k, v))
    both = torch.zeros((5, 2, 2, 64), dtype=torch.bfloat16)

    class Passed(Exception):
        pass

    def passed(*_):
        raise Passed
    cache._list = passed                                            # the next step: the arguments were taken
    for k, v in ((both[:, 0], both[:, 1]), (both[:, :, 0], both[:, :, 1]), (x[:4], x[4:])):
        with pytest.raises(Passed):
            cache.read(0, seqs, cu, out=(k, v))
