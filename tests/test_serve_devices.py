"""Serving calls on tensors of a device that is not the current one, on the CPU: a library in the native one's place notes
which device is current when it is called, and stand-ins take the tensors' places."""

import itertools
import types

import pytest


class Tensor:
    """Shape, type and place of a tensor on cuda:1."""
    is_cuda = True
    made = itertools.count(1)

    def __init__(self, *shape, dtype=None):
        import torch
        self.shape, self.dtype, self.device = torch.Size(shape), dtype or torch.bfloat16, torch.device("cuda", 1)
        self.at = next(self.made) << 20

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        s = [1]
        for n in reversed(self.shape[1:]):
            s.insert(0, s[0] * n)
        return tuple(s) if i is None else s[i]

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.at

    def element_size(self):
        return self.dtype.itemsize


@pytest.fixture
def world(monkeypatch):
    """current: the current device; calls: (entry, current device, stream) of every launch."""
    import torch
    from tensorpack_amd import _native, attention, cache, device, sampling
    w = types.SimpleNamespace(current=0, calls=[])

    class Guard:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.was, w.current = w.current, self.index

        def __exit__(self, *a):
            w.current = self.was

    class Library:
        def __getattr__(self, name):
            if name.endswith("_bytes"):
                return lambda *a: 64
            return lambda *a: w.calls.append((name, w.current, a[-1])) or 0
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: w.current, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(_native, "hip_lib", Library)
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **k: empty(*a, **k))
    for m in (attention, cache, sampling):
        monkeypatch.setattr(m, "raw_stream", lambda index: 1000 + index)
    for m in (attention, sampling):
        monkeypatch.setattr(m, "stream_workspace", lambda index, stream, need: w.calls.append(("workspace", w.current, stream)) or Tensor(need))
    for m in (attention, cache):
        monkeypatch.setattr(m, "_int32", lambda name, x, n, dev: 0x2000)
    w.cache = object.__new__(cache.PagedCache)
    w.cache.__dict__.update(device=torch.device("cuda", 1), dtype=torch.bfloat16, lib=Library(), desc_ref=None, n_layers=2, n_kv_heads=2,
                            head_dim=64, max_seqs=8, desc=types.SimpleNamespace(dtype=1))
    return w


def test_launches_go_to_the_tensors_device(world):
    import torch
    from tensorpack_amd.attention import cached_attention, prompt_attention
    from tensorpack_amd.sampling import verify_drafts
    i32, f32 = dict(dtype=torch.int32), dict(dtype=torch.float32)
    two, cu = Tensor(2, **i32), Tensor(3, **i32)
    prompt_attention(Tensor(8, 4, 64), Tensor(8, 2, 64), Tensor(8, 2, 64), cu, out=Tensor(8, 4, 64))
    cached_attention(Tensor(2, 1, 4, 64), world.cache, 0, two, out=Tensor(2, 1, 4, 64))
    verify_drafts(Tensor(2, 3, **i32), Tensor(2, 4, 100, **f32), Tensor(2, 3, 100, **f32), Tensor(2, 3, **f32), Tensor(2, 100, **f32))
    c = world.cache
    c.extend(two, two)
    c.append(0, Tensor(5, 2, 64), Tensor(5, 2, 64), two, cu)
    c.fork(two, two)
    c.truncate(two, two)
    c.free(two)
    c.compact()
    launches = [x for x in world.calls if x[0] != "workspace"]
    assert [x[0] for x in launches] == ["mtc_prompt_attention", "mtc_cached_attention", "mtc_verify_drafts", "mtc_cache_extend",
                                        "mtc_cache_append", "mtc_cache_fork", "mtc_cache_truncate", "mtc_cache_truncate", "mtc_cache_compact"]
    assert all(x[1:] == (1, 1001) for x in world.calls), world.calls
    assert len(world.calls) == len(launches) + 3 and world.current == 0


def test_append_holds_its_copies_until_the_launch(world, monkeypatch):
    """K and V that have to be copied: both copies live when the library is called (another thread could get the
    memory of a released one on the same stream)."""
    import weakref
    from tensorpack_amd import cache
    copies, alive = [], []

    def copy(x):
        y = Tensor(*x.shape)
        copies.append(weakref.ref(y))
        return y
    monkeypatch.setattr(cache, "_copy", copy)
    world.cache.lib.__class__.mtc_cache_append = lambda self, *a: alive.extend(r() is not None for r in copies) or 0
    k, v = Tensor(5, 2, 64), Tensor(5, 2, 64)
    k.data_ptr = v.data_ptr = lambda: 0x100002
    import torch
    world.cache.append(0, k, v, Tensor(2, dtype=torch.int32), Tensor(3, dtype=torch.int32))
    assert alive == [True, True]
