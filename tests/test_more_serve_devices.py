"""Rotary positions, reading an 8-bit cache, reordering and the beam step on tensors of a device that is not the current one, on the
CPU (see test_serve_devices)."""

import types

from test_serve_devices import Tensor, world                     # noqa: F401  (a fixture)


def test_launches_go_to_the_tensors_device(world, monkeypatch):  # noqa: F811
    import torch
    from tensorpack_amd import _abi, cache, rotary, sampling
    monkeypatch.setattr(rotary, "raw_stream", lambda index: 1000 + index)
    monkeypatch.setattr(rotary, "_int32", lambda name, x, n, dev: 0x2000)
    monkeypatch.setattr(torch, "empty_like", lambda x, **k: Tensor(*x.shape, dtype=x.dtype))
    monkeypatch.setattr(Tensor, "contiguous", lambda self: self, raising=False)
    i32, f32 = dict(dtype=torch.int32), dict(dtype=torch.float32)
    turn = types.SimpleNamespace(device=torch.device("cuda", 1), dim=64, interleaved=False, amplitude=1.0, turns_at=0x3000)
    rotary.apply_rotary(turn, Tensor(5, 4, 64), Tensor(5, 2, 64), Tensor(5, **i32))
    rotary.apply_rotary(turn, Tensor(5, 4, 64), None, Tensor(5, **i32), out=(Tensor(5, 4, 64), None))
    c = object.__new__(cache.QuantizedCache)
    c.__dict__.update(world.cache.__dict__, desc=types.SimpleNamespace(dtype=1 | _abi.CACHE_CODES8))
    two, cu = Tensor(2, **i32), Tensor(3, **i32)
    c.append(0, Tensor(5, 2, 64), Tensor(5, 2, 64), two, cu)
    c.read(0, two, cu, out=(Tensor(5, 2, 64), Tensor(5, 2, 64)))
    c.read(0, two, cu, 5)
    c.reorder(two, two)
    sampling.beam_select(Tensor(2, 3, 100, **f32), Tensor(2, 3, **f32))
    launches = [x for x in world.calls if x[0] != "workspace"]
    assert [x[0] for x in launches] == ["mtc_rotary", "mtc_rotary", "mtc_cache_append", "mtc_cache_read", "mtc_cache_read", "mtc_cache_reorder", "mtc_beam_select"]
    assert all(x[1:] == (1, 1001) for x in world.calls), world.calls
    assert len(world.calls) == len(launches) + 1 and world.current == 0


def test_copies_live_until_the_launch(world, monkeypatch):       # noqa: F811
    """q and k that have to be copied: both copies live when the library is called."""
    import weakref
    import torch
    from tensorpack_amd import _native, rotary
    monkeypatch.setattr(rotary, "raw_stream", lambda index: 1000 + index)
    monkeypatch.setattr(rotary, "_int32", lambda name, x, n, dev: 0x2000)
    copies, alive = [], []

    def copy(x):
        y = Tensor(*x.shape)
        copies.append(weakref.ref(y))
        return y
    monkeypatch.setattr(rotary, "_copy", copy)
    lib = types.SimpleNamespace(mtc_rotary=lambda *a: alive.extend(r() is not None for r in copies) or 0)
    monkeypatch.setattr(_native, "hip_lib", lambda: lib)
    q, k = Tensor(5, 4, 64), Tensor(5, 2, 64)
    q.data_ptr = k.data_ptr = lambda: 0x100002
    turn = types.SimpleNamespace(device=torch.device("cuda", 1), dim=64, interleaved=False, amplitude=1.0, turns_at=0x3000)
    rotary.apply_rotary(turn, q, k, Tensor(5, dtype=torch.int32), out=(Tensor(5, 4, 64), Tensor(5, 2, 64)))
    assert alive == [True, True]
