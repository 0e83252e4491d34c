"""verify_drafts against its rule in Python and 64 bits. Tokens and counts are compared for equality: the inputs are random
fp32 / 16-bit numbers, whose products have no ties within fp32's rounding, except where a test makes exact ties."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _inputs(B, K, V, dtype, seed, close=0.5, index=None):
    import torch
    g = torch.Generator().manual_seed(seed)
    dt = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    logits = torch.randn((B, K + 1, V), generator=g) * 2
    p = torch.softmax(logits, -1).to(dt)
    q = torch.softmax(logits[:, :K] + close * torch.randn((B, K, V), generator=g), -1)
    race = 1.0 / torch.empty((B, K, V)).exponential_(generator=g).clamp_min(1e-20)
    drafts = (q * race).argmax(-1).to(index or torch.int32)
    noise = 1.0 / torch.empty((B, V)).exponential_(generator=g).clamp_min(1e-20)
    return drafts, p, q.to(dt), torch.rand((B, K), generator=g), noise


def _plain(drafts, p, q, u, noise, n_drafts=None):
    d, p, q, u, noise = (t.cpu().numpy() if t.dtype.is_floating_point is False else t.double().cpu().numpy()
                         for t in (drafts, p, q, u, noise))
    B, K = d.shape
    tokens, counts = np.full((B, K + 1), -1), np.zeros(B, int)
    for b in range(B):
        k = K if n_drafts is None else min(max(n_drafts[b], 0), K)
        n = 0
        while n < k and 0 <= d[b, n] < p.shape[2] and u[b, n] * q[b, n, d[b, n]] < p[b, n, d[b, n]]:
            n += 1
        w = p[b, n]
        if n < k:
            rest = np.maximum(w - q[b, n], 0)
            w = rest if (rest > 0).any() else w
        score = np.where(w > 0, w * noise[b], -1.0)
        tokens[b, :n] = d[b, :n]
        tokens[b, n] = int(score.argmax()) if score.max() >= 0 else -1
        counts[b] = n
    return tokens, counts


def _check(got, want):
    assert np.array_equal(got[0].cpu().numpy(), want[0])
    assert np.array_equal(got[1].cpu().numpy(), want[1])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 500), (3, 7, 4099), (40, 3, 1001), (2, 64, 257), (1, 2, 70001), (5, 0, 777)])
def test_verify(gpu, dtype, B, K, V):
    import torch
    from tensorpack_amd.sampling import verify_drafts
    print("verify", dtype, B, K, V, flush=True)
    seen = set()
    for seed, close in ((0, 0.5), (1, 0.1), (2, 2.0)):
        x = _inputs(B, K, V, dtype, 10 * V + seed, close, torch.int64 if seed else None)
        y = [t.to(gpu) for t in x]
        got = verify_drafts(*y)
        assert got[0].dtype == x[0].dtype
        want = _plain(*x)
        _check(got, want)
        n = [(i * 5 + seed) % (K + 3) - 1 for i in range(B)]                      # below 0 and above K too
        _check(verify_drafts(*y, n_drafts=torch.tensor(n, dtype=torch.int32, device=gpu)), _plain(*x, n_drafts=n))
        seen |= set(want[1].tolist())
    assert len(seen) > 1 or K == 0 or V == 1


def test_verify_distribution(gpu):
    # the tokens' distribution is the target's: chi-square over 200000 one-draft sequences, 31 degrees of freedom
    import torch
    from tensorpack_amd.sampling import verify_drafts
    B, V = 50000, 32
    g = torch.Generator().manual_seed(3)
    p, q = torch.softmax(torch.randn(V, generator=g), 0), torch.softmax(torch.randn(V, generator=g), 0)
    count = torch.zeros(V)
    for _ in range(4):
        drafts = torch.multinomial(q, B, replacement=True, generator=g).int()[:, None]
        noise = 1.0 / torch.empty((B, V)).exponential_(generator=g).clamp_min(1e-20)
        u = torch.rand((B, 1), generator=g)
        tokens, _ = verify_drafts(*(t.to(gpu) for t in (drafts, p.expand(B, 2, V), q.expand(B, 1, V), u, noise)))
        count += torch.bincount(tokens[:, 0].cpu().long(), minlength=V)
    n = count.sum()
    chi = float(((count - n * p) ** 2 / (n * p)).sum())
    assert chi < 31 + 6 * (2 * 31) ** 0.5                                         # six standard deviations


def test_verify_edges(gpu):
    import torch
    from tensorpack_amd.sampling import verify_drafts
    V = 5000
    drafts, p, q, u, noise = (t.to(gpu) for t in _inputs(6, 2, V, "fp32", 7))
    q[0, 0], drafts[0, 0], u[0, 0] = p[0, 0], 17, 1.0            # nothing is left of p - q: the next token comes from p
    p[1, 0, :] = 0                                               # nothing at all: -1
    drafts[2, 0], drafts[3, 0] = V, -1                           # outside the vocabulary: rejected
    p[4, 0, int(drafts[4, 0])], q[4, 0, int(drafts[4, 0])] = float("nan"), 0.1    # a NaN is not accepted and not drawn
    noise[5] = 1.0
    p[5, 0], q[5, 0], u[5, 0] = 0.25, 0.0, 0.0
    p[5, 1], q[5, 1], u[5, 1] = 0.25, 0.0, 0.0
    p[5, 2] = 0.125
    p[5, 2, 4321], p[5, 2, 1234], p[5, 2, 3000] = 0.5, 0.5, 0.5  # exact ties: the first index
    tokens, n = (t.cpu().numpy() for t in verify_drafts(drafts, p, q, u, noise))
    w = (p[0, 0].double() * noise[0].double()).cpu().numpy()
    assert n[0] == 0 and tokens[0, 0] == w.argmax()
    assert n[1] == 0 and tokens[1].tolist() == [-1, -1, -1]
    assert n[2] == 0 and n[3] == 0 and n[4] == 0 and 0 <= tokens[4, 0] < V and tokens[4, 0] != int(drafts[4, 0])
    assert n[5] == 2 and tokens[5].tolist() == drafts[5].tolist() + [1234]


def test_verify_views_stream_and_graph(gpu):
    import torch
    from tensorpack_amd.sampling import verify_drafts
    B, K, V = 9, 3, 2051
    x = [t.to(gpu) for t in _inputs(B, K, V, "bf16", 5)]
    want = verify_drafts(*x)
    wide = torch.zeros((B, K + 4, V + 5), dtype=torch.bfloat16, device=gpu)
    p, q = wide[:, :K + 1, 3:3 + V], wide.clone()[:, 1:1 + K, 2:2 + V]
    p.copy_(x[1])
    q.copy_(x[2])
    noise = torch.zeros((B, V + 1), device=gpu)[:, 1:]
    noise.copy_(x[4])
    got = verify_drafts(x[0], p, q, x[3], noise)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = verify_drafts(x[0].t().contiguous().t(), x[1].transpose(1, 2).contiguous().transpose(1, 2), x[2], x[3], x[4])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = verify_drafts(*x)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = verify_drafts(*x)
    for i in range(3):
        x[3].uniform_()
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, verify_drafts(*x)))


def test_verify_refusals(gpu):
    import torch
    from tensorpack_amd.sampling import verify_drafts
    d, p, q, u, e = (t.to(gpu) for t in _inputs(2, 3, 50, "fp32", 1))
    for args in ((d.float(), p, q, u, e), (d, p, q.half(), u, e), (d, p.double(), q.double(), u, e), (d, p[:, :3], q, u, e),
                 (d, p, q[:, :2], u, e), (d, p, q, u.double(), e), (d, p, q, u, e[:1]), (d, p, q, u, e.half()), (d[0], p, q, u, e),
                 (d, p[..., :49], q, u, e), (d.cpu(), p, q, u, e)):
        with pytest.raises(ValueError):
            verify_drafts(*args)
    for n in (torch.zeros(2, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu)):
        with pytest.raises(ValueError):
            verify_drafts(d, p, q, u, e, n_drafts=n)
    with pytest.raises(ValueError):
        verify_drafts(d.expand(2, 3).repeat(1, 22), p[:, :1].expand(2, 67, 50), q[:, :1].expand(2, 66, 50), u.repeat(1, 22), e)
    assert verify_drafts(d[:0], p[:0], q[:0], u[:0], e[:0])[0].shape == (0, 4)
