"""apply_rotary against the turn in 64 bits (angles by Python's integers where positions are far).

Tolerances. The kernel's sine and cosine, times the amplitude, are off by less than 2e-7 of the amplitude: the angle within an
eighth of a turn is rounded twice (each 2^-24 of at most 0.79: 9.4e-8), the series by its last sum (3e-8, the others less) and
its first term left out (2e-9), the product with the amplitude once (6e-8). A product of them with x and y, and the sum, in fp32: |error| <= a (|x| + |y|) (2e-7 + 2 * 2^-24),
and one rounding of the result to its type, half a step: eps / 2 of it (f16 below 2^-14: half of 2^-24)."""

import math
from fractions import Fraction

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _want(x, positions, freqs, rd, interleaved, amplitude):
    """(turned in 64 bits, |x| + |y| of each element's pair)."""
    from tensorpack_amd.rotary import _PI
    y, size = x.astype(np.float64), np.zeros(x.shape)
    for i, f in enumerate(freqs):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rd // 2)
        turns = [float(int(p) * Fraction(f) / (2 * _PI) % 1) for p in positions]
        t = 2 * math.pi * np.array(turns)[:, None]
        u, v = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
        y[..., a], y[..., b] = amplitude * (u * np.cos(t) - v * np.sin(t)), amplitude * (u * np.sin(t) + v * np.cos(t))
        size[..., a] = size[..., b] = abs(amplitude) * (np.abs(u) + np.abs(v))
    return y, size


def _check(got, x, positions, rotary):
    import torch
    want, size = _want(x.double().cpu().numpy(), positions, rotary.frequencies, rotary.dim, rotary.interleaved, rotary.amplitude)
    eps = torch.finfo(x.dtype).eps
    least = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= size * (2e-7 + 2 ** -23) * 1.01 + np.maximum(eps / 2 * np.abs(want) * 1.01, least)).all(), float(err.max())
    assert torch.equal(got[..., rotary.dim:], x[..., rotary.dim:])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,kv,dim,rd", [(1, 14, 2, 64, 64), (5, 4, 4, 128, 64), (33, 3, 1, 40, 40), (7, 2, 1, 40, 20), (9, 5, 2, 40, 10),
                                                  (3, 1, 1, 8, 2), (300, 32, 8, 128, 128), (2500, 16, 16, 80, 32), (4, 2, 1, 256, 48)])
def test_against_64_bits(gpu, dtype, interleaved, rows, heads, kv, dim, rd):
    import torch
    from tensorpack_amd.rotary import Rotary, apply_rotary
    g = torch.Generator().manual_seed(rows * 7 + dim)
    q, k = (torch.randn((rows, h, dim), generator=g).to(getattr(torch, dtype)).to(gpu) for h in (heads, kv))
    positions = torch.randint(0, 5000, (rows,), generator=g, dtype=torch.int32)
    r = Rotary(rd, interleaved=interleaved, amplitude=1.25 if rd == 64 else 1.0, device=gpu)
    a, b = apply_rotary(r, q, k, positions.to(gpu))
    keep = slice(0, 200)                                            # the oracle is slow
    _check(a[keep], q[keep], positions.tolist()[keep], r)
    _check(b[keep], k[keep], positions.tolist()[keep], r)
    _check(a[-5:], q[-5:], positions.tolist()[-5:], r)


def test_far_and_negative_positions(gpu):
    import torch
    from tensorpack_amd.rotary import Rotary, apply_rotary
    p = [0, 1, -1, 4095, 1 << 20, (1 << 20) + 1, 2 ** 31 - 1, -2 ** 31, 1234567890, -987654321]
    for kw in ({}, {"factor": 8.0, "original": 8192}, {"factor": 3.5}, {"frequencies": [0.0, 7.5, math.pi, 1e-9] * 8}):
        r = Rotary(64, device=gpu, **kw)
        q = torch.randn((len(p), 3, 64), generator=torch.Generator().manual_seed(1)).to(gpu)
        a, b = apply_rotary(r, q, None, torch.tensor(p, dtype=torch.int32, device=gpu))
        assert b is None
        _check(a, q, p, r)


def test_views_in_place_and_copies(gpu):
    """Views of one product's result; results into the inputs themselves; inputs that must be copied first; other
    memory of the buffers stays as it was."""
    import torch
    from tensorpack_amd.rotary import Rotary, apply_rotary
    r = Rotary(32, device=gpu)
    pos = torch.arange(50, 57, dtype=torch.int32, device=gpu)
    x = torch.randn((9, (4 + 2 + 2) * 64), generator=torch.Generator().manual_seed(2)).bfloat16().to(gpu)
    q, k, v = (t.unflatten(1, (-1, 64))[1:8] for t in x.split([256, 128, 128], dim=1))
    want = apply_rotary(r, q.contiguous(), k.contiguous(), pos)
    got = apply_rotary(r, q, k, pos)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for odd in (q[:, :, 1:33], torch.randn((7, 64, 4), device=gpu).bfloat16().transpose(1, 2), q[:, ::3], q[:1].expand(7, 4, 64)):
        assert torch.equal(apply_rotary(r, odd, None, pos)[0], apply_rotary(r, odd.contiguous(), None, pos)[0])
    before = x.clone()
    apply_rotary(r, q, k, pos, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    q.copy_(before[1:8, :256].unflatten(1, (-1, 64)))
    k.copy_(before[1:8, 256:384].unflatten(1, (-1, 64)))
    assert torch.equal(x, before)
    by_heads = torch.empty((4, 7, 64), dtype=torch.bfloat16, device=gpu).transpose(0, 1)
    assert torch.equal(apply_rotary(r, q, None, pos, out=(by_heads, None))[0], want[0])


def test_rows_far_apart(gpu):
    """Rows 2 GiB apart, in and out: offsets pass 32 bits."""
    import torch
    from tensorpack_amd.rotary import Rotary, apply_rotary
    r = Rotary(64, device=gpu)
    pos = torch.tensor([3, 70, 1000, 5], dtype=torch.int32, device=gpu)
    buf = torch.empty((3 << 30) + 4096, dtype=torch.bfloat16, device=gpu)
    far = lambda at, h: buf.as_strided((4, h, 64), (1 << 30, 64, 1), at)
    near = [torch.randn((4, h, 64), generator=torch.Generator().manual_seed(h)).bfloat16().to(gpu) for h in (4, 2)]
    q, k, to = far(0, 4), far(512, 2), (far(1024, 4), far(2048, 2))
    q.copy_(near[0])
    k.copy_(near[1])
    apply_rotary(r, q, k, pos, out=to)
    assert all(torch.equal(a, b) for a, b in zip(to, apply_rotary(r, *near, pos)))
    assert torch.equal(q, near[0]) and torch.equal(k, near[1])


def test_nothing_to_do_and_infinities(gpu):
    import torch
    from tensorpack_amd.rotary import Rotary, apply_rotary
    r = Rotary(8, device=gpu)
    none = torch.zeros((0,), dtype=torch.int32, device=gpu)
    a, b = apply_rotary(r, torch.zeros((0, 2, 16), device=gpu), torch.zeros((0, 1, 16), device=gpu), none)
    assert a.shape == (0, 2, 16) and b.shape == (0, 1, 16)
    q = torch.ones((2, 1, 16), device=gpu)
    q[0, 0, 3] = math.nan
    q[0, 0, 9] = math.inf
    a, _ = apply_rotary(r, q, None, torch.tensor([5, 5], dtype=torch.int32, device=gpu))
    assert torch.isnan(a[0, 0, [3, 7]]).all() and torch.isfinite(a[0, 0, [0, 1, 2, 4, 5, 6, 8]]).all()       # its own pair only
    assert torch.equal(a[0, 0, [0, 1, 2, 4, 5, 6]], a[1, 0, [0, 1, 2, 4, 5, 6]]) and a[0, 0, 9] == math.inf


def test_capture_and_streams(gpu):
    import torch
    from tensorpack_amd.rotary import Rotary, apply_rotary
    r = Rotary(64, device=gpu)
    q, k = torch.randn((6, 4, 64), device=gpu), torch.randn((6, 2, 64), device=gpu)
    pos = torch.arange(6, dtype=torch.int32, device=gpu)
    out = (torch.empty_like(q), torch.empty_like(k))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apply_rotary(r, q, k, pos, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        apply_rotary(r, q, k, pos, out=out)
        pos.add_(1)
    for step in range(3):
        at = pos.clone()
        graph.replay()
        want = apply_rotary(r, q, k, at)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals(gpu):
    import torch
    from tensorpack_amd.rotary import Rotary, apply_rotary, rotary_frequencies
    r = Rotary(64, device=gpu)
    q, pos = torch.zeros((4, 2, 64), device=gpu), torch.zeros(4, dtype=torch.int32, device=gpu)
    other = q.clone()
    for bad in (dict(q=q.double()), dict(q=q[0]), dict(q=q[..., :60]), dict(q=q[..., :32]), dict(k=q.half()), dict(k=q[:3]),
                dict(positions=pos.long()), dict(positions=pos[:3]), dict(positions=pos.cpu()), dict(q=q.cpu()),
                dict(out=(q, q)), dict(out=(q[..., 1:], None)), dict(out=(q[:1].expand(4, 2, 64), None)),
                dict(k=q.clone(), out=(other, other)), dict(k=other, out=(other, torch.empty_like(q))), dict(k=other, out=(torch.empty_like(q), q)),
                dict(out=(torch.zeros((4, 130), device=gpu)[:, :128].unflatten(1, (2, 64)), None))):
        kw = {**dict(q=q, k=None, positions=pos), **bad}
        with pytest.raises(ValueError):
            apply_rotary(r, **kw)
    for bad in (dict(dim=63), dict(dim=0), dict(dim=64, base=-1.0), dict(dim=64, factor=0.5), dict(dim=64, original=0), dict(dim=64, original=9, ramp=(2.0, 2.0)),
                dict(dim=64, frequencies=[1.0] * 31), dict(dim=4, frequencies=[1.0, math.inf]), dict(dim=64, amplitude=math.nan)):
        with pytest.raises(ValueError):
            Rotary(device=gpu, **bad)
    assert rotary_frequencies(4, base=100.0) == [1.0, 0.1]
