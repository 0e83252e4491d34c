"""Calls that hand partial results on from kernel to kernel: what overlaps in time has workspaces of its own. Equality only."""

import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _ints(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _calls(dev, seed):
    """Callables, one per operator with a workspace, on inputs of their own."""
    import torch
    from tensorpack_amd.attention import cached_attention, prompt_attention
    from tensorpack_amd.cache import PagedCache
    from tensorpack_amd.sampling import verify_drafts
    g = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device=dev).bfloat16()
    cache = PagedCache(80, 1, 2, 64, max_seqs=2, max_pages=40, device=dev)
    cache.pool.copy_(normal(*cache.pool.shape))
    cache.extend(_ints([0, 1], dev), _ints([600, 30 + seed], dev))
    q, k, v = normal(2, 1, 4, 64), normal(3000, 2, 64), normal(3000, 2, 64)
    few, cq, ck, seqs = normal(9, 4, 64), _ints([0, 9], dev), _ints([0, 3000], dev), _ints([0, 1], dev)
    p = torch.softmax(torch.randn((3, 4, 5000), generator=g, device=dev), -1)
    d = torch.softmax(torch.randn((3, 3, 5000), generator=g, device=dev), -1)
    drafts, u = d.argmax(-1).int(), torch.rand((3, 3), generator=g, device=dev)
    noise = 1.0 / torch.empty((3, 5000), device=dev).exponential_(generator=g)
    return [lambda: cached_attention(q, cache, 0, seqs), lambda: prompt_attention(few, k, v, cq, ck),
            lambda: verify_drafts(drafts, p, d, u, noise)[0]]


@pytest.fixture
def taken(monkeypatch):
    """(thread, first byte, past the last byte) of every workspace that a serving call takes."""
    from tensorpack_amd import attention, device, sampling
    out = []

    def record(index, stream, need):
        t = device.stream_workspace(index, stream, need)
        out.append((threading.get_ident(), t.data_ptr(), t.data_ptr() + need))
        return t
    monkeypatch.setattr(attention, "stream_workspace", record)
    monkeypatch.setattr(sampling, "stream_workspace", record)
    return out


def _apart(a, b):
    return all(x[2] <= y[1] or y[2] <= x[1] for x in a for y in b)


def test_threads_on_one_stream(gpu, taken):
    import torch
    want = [[f() for f in _calls(gpu, s)] for s in (1, 2)]
    torch.cuda.synchronize()
    taken.clear()
    got, errs, ready = [None, None], [], threading.Barrier(2)

    def run(i):
        try:
            calls = _calls(gpu, i + 1)
            ready.wait()
            got[i] = [[f() for f in calls] for _ in range(30)]
            ready.wait()                                         # neither thread's buffers are released before both are done
        except Exception as e:                                   # reported below
            errs.append(e)
            ready.abort()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errs, errs
    assert all(torch.equal(x, y) for i in range(2) for row in got[i] for x, y in zip(row, want[i]))
    ids = sorted({t for t, _, _ in taken})
    assert len(ids) == 2 and len(taken) == 2 * 30 * 3
    assert _apart([x for x in taken if x[0] == ids[0]], [x for x in taken if x[0] == ids[1]])


def test_graphs_replayed_side_by_side(gpu, taken):
    import torch
    calls = [_calls(gpu, s) for s in (1, 2)]
    want = [[f() for f in c] for c in calls]
    graphs, outs, spans = [], [], []
    for c in calls:
        taken.clear()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):                                # both on the stream that torch captures on by default
            outs.append([f() for f in c])
        graphs.append(g)
        spans.append(list(taken))
    assert len(spans[0]) == len(spans[1]) == 3 and _apart(*spans)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for a, b in zip(outs, want) for x, y in zip(a, b))
        [f() for f in calls[0]]                                  # eager calls between the replays keep out of their memory


def test_a_captured_prefill_keeps_out_of_eager_calls(gpu):
    """A product that stages and splits, captured, then an eager one that needs more workspace on the same stream."""
    import torch
    from tensorpack_amd.kernels.gemm import MTCMatrix
    from tensorpack_amd.core.quadtree import QuadtreeRD
    rng = np.random.RandomState(0)
    m = MTCMatrix.from_quadtree(QuadtreeRD((rng.randn(512, 256) * 0.05).astype(np.float32), None, (32, 16, 8, 4)).select(4.0))
    t = m.device_tiles(gpu)
    X, big = (torch.from_numpy(rng.randn(n, 512).astype(np.float32)).to(gpu) for n in (300, 2000))
    want, large = t.gemm_bf16(X), t.gemm_bf16(big)
    g, Y, s = torch.cuda.CUDAGraph(), torch.empty_like(want), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        t.gemm_bf16(X, out=Y)
    for _ in range(4):
        Y.zero_()
        g.replay()
        with torch.cuda.stream(s):
            s.wait_stream(torch.cuda.default_stream())
            assert torch.equal(t.gemm_bf16(big), large)
        torch.cuda.synchronize()
        assert torch.equal(Y, want)


def test_a_captured_decode_keeps_its_workspace(gpu):
    """A split-K decode of 2 rows captured, then calls of other row counts on the same stream, whose workspaces have other sizes:
    the graph's stays where it was."""
    import torch
    from tensorpack_amd.core.quadtree import QuadtreeRD
    from tensorpack_amd.kernels.gemm import MTCMatrix
    rng = np.random.RandomState(1)
    m = MTCMatrix.from_quadtree(QuadtreeRD((rng.randn(512, 256) * 0.05).astype(np.float32), None, (32, 16, 8, 4)).select(4.0))
    ds, s = m.device_stream(64, gpu, 2), torch.cuda.Stream()
    X = {n: torch.from_numpy(rng.randn(n, 512).astype(np.float32)).to(gpu) for n in (1, 2, 16)}
    want = {n: ds.gemv_f32(x) for n, x in X.items()}
    Y, g = torch.empty_like(want[2]), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        ds.gemv_f32(X[2], out=Y)
        held = ds.workspace(2)[0]
    sizes = {int(ds.lib.mtc_gemv_workspace_bytes(ds.desc, n)) for n in X}
    assert len(sizes) > 1 and held is not None
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        ds.gemv_f32(X[2], out=Y)
    for n in (16, 1, 16):
        with torch.cuda.stream(s):
            assert torch.equal(ds.gemv_f32(X[n]), want[n])
            assert ds.workspace(2)[0] is held
        torch.cuda.synchronize()
        Y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(Y, want[2])


@pytest.mark.parametrize("rows", [3, 16])
def test_decodes_of_two_threads_on_one_stream(gpu, rows):
    """Split-K decode (counters) and, from 5 rows, X laid out by a launch of its own: the threads' workspaces are apart."""
    import torch
    from tensorpack_amd.core.quadtree import QuadtreeRD
    from tensorpack_amd.kernels.gemm import MTCMatrix
    rng = np.random.RandomState(2)
    m = MTCMatrix.from_quadtree(QuadtreeRD((rng.randn(512, 256) * 0.05).astype(np.float32), None, (32, 16, 8, 4)).select(4.0))
    ds = m.device_stream(64, gpu, rows)
    X = [torch.from_numpy(rng.randn(rows, 512).astype(np.float32)).to(gpu) for _ in range(2)]
    want = [ds.gemv_f32(x) for x in X]
    torch.cuda.synchronize()
    got, spans, errs, ready = [None, None], [None, None], [], threading.Barrier(2)

    def run(i):
        try:
            ready.wait()
            got[i] = [ds.gemv_f32(X[i]) for _ in range(50)]
            ws, n = ds.workspace(rows)
            spans[i] = [(0, ws.data_ptr(), ws.data_ptr() + n)]
            ready.wait()
        except Exception as e:                                   # reported below
            errs.append(e)
            ready.abort()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errs, errs
    assert _apart(*spans)
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
