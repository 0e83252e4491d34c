"""beam_select against its definition in 64 bits. Tokens and parents are compared for equality: the inputs' scores lie further apart
than the kernel's error, or are equal for a reason that the kernel shares (equal logits of one beam), which the test checks.

Tolerance of the scores: exponentials (two roundings and the hardware's, 3 * 2^-24 of each) and their fp32 sums (64 terms in a lane,
one after another, and 6 sums over lanes: up to 70 * 2^-24) give the logarithm an error below 80 * 2^-24 = 4.8e-6; the result is
rounded once."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LOG_ERROR = 80 * 2.0 ** -24
MANY = [(500, 1, 0), (500, 16, 0), (500, 31, 0), (500, 33, 0), (500, 64, 0), (9000, 1, 0), (9000, 16, 0), (9000, 31, 0),
        (9000, 33, 0), (9000, 64, 0), (32000, 1, 0), (32000, 16, 0), (32000, 31, 0), (32000, 33, 0), (32000, 64, 0)]                  # vocabulary, beams that go on, seed


def _ints(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _want(logits, scores, n, done=None, pad=0):
    """Lists of (score, token, row) per prompt."""
    x = logits.double().cpu().numpy()
    B, W, V = x.shape
    s = scores.double().cpu().numpy()
    out = []
    for b in range(B):
        found = []
        for w in range(W):
            if done is not None and done[b][w]:
                found.append((s[b, w], w, 0, pad))
                continue
            top = x[b, w].max()
            if not np.isfinite(top):
                continue
            y = s[b, w] + x[b, w] - (top + math.log(np.exp(x[b, w] - top).sum()))
            for v in np.argsort(-y, kind="stable")[:n]:
                found.append((y[v], w, int(v), int(v)))
        found = sorted((f for f in found if f[0] > -np.inf), key=lambda f: (-f[0], f[1], f[2]))
        assert all(a[0] == c[0] and a[1] == c[1] or a[0] - c[0] > 4 * LOG_ERROR or a[1] == c[1] for a, c in zip(found[:n], found[1:n + 1]))
        rows = [(f[0], f[3], b * W + f[1]) for f in found[:n]]
        out.append(rows + [(-np.inf, -1, b * W + min(k, W - 1)) for k in range(len(rows), n)])
    return out


def _check(got, want):
    scores, tokens, parents = (t.cpu().numpy() for t in got)
    for b, rows in enumerate(want):
        assert [int(x) for x in tokens[b]] == [r[1] for r in rows], b
        assert [int(x) for x in parents[b]] == [r[2] for r in rows], b
        for x, (s, _, _) in zip(scores[b], rows):
            assert (x == s) if not math.isfinite(s) else abs(float(x) - s) <= LOG_ERROR + 2.0 ** -24 * abs(s), (b, x, s)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("B,W,V,n", [(1, 4, 32000, 4), (3, 1, 7, 1), (2, 5, 513, 9), (7, 3, 4096, 6), (1, 16, 128003, 16), (2, 64, 700, 64), (5, 2, 50257, 1),
                                     (9, 8, 128003, 8), (1, 2, 1, 5)])
def test_against_64_bits(gpu, dtype, B, W, V, n):
    import torch
    from tensorpack_amd.sampling import beam_select
    print("beam", dtype, B, W, V, n, flush=True)
    g = torch.Generator().manual_seed(V + n)
    logits = (torch.randn((B, W, V), generator=g) * 3).to(getattr(torch, dtype)).to(gpu)
    scores = (-30 * torch.rand((B, 1), generator=g) - 4 * torch.rand((B, W), generator=g)).to(gpu)
    got = beam_select(logits, scores, n=n)
    assert got[0].shape == got[1].shape == got[2].shape == (B, n) and got[1].dtype == got[2].dtype == torch.int32
    _check(got, _want(logits, scores, n))
    again = beam_select(logits, scores, n=n)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("V", [100, 5000, 700000])
def test_ended_beams_and_first_steps(gpu, V):
    import torch
    from tensorpack_amd.sampling import beam_select
    g = torch.Generator().manual_seed(1)
    logits = (torch.randn((4, 4, V), generator=g) * 2).to(gpu)
    scores = torch.tensor([[0.0] + [-math.inf] * 3, [-9.0, -2.0, -30.0, -1.0], [-1.0, -2.0, -3.0, -4.0], [-math.inf] * 4], device=gpu)
    done = [[False] * 4, [False, True, False, True], [True] * 4, [True, False, True, False]]
    logits[1, 1] = math.nan                                      # an ended beam's logits have no part
    got = beam_select(logits, scores, done=torch.tensor(done, device=gpu), pad=77)
    _check(got, _want(logits, scores, 4, done, 77))
    assert got[2][0].tolist() == [0, 0, 0, 0] and got[1][2].tolist() == [77] * 4
    many = beam_select(logits, scores, n=9, done=torch.tensor(done, device=gpu), pad=-5)
    _check(many, _want(logits, scores, 9, done, -5))
    assert many[1][3].tolist() == [-1] * 9 and many[0][2][4:].tolist() == [-math.inf] * 5


def _many(V, live, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn((2, 64, V), generator=g) * 3 + 100
    scores = torch.full((2, 64), -math.inf)
    scores[0, :live] = torch.randn(live, generator=g)
    scores[1, 64 - live:] = torch.randn(live, generator=g) * 100
    logits[1, 63, 5:] = -math.inf
    logits[0, 0, 70:] = -math.inf
    if live > 16:
        logits[0, 7] = math.nan
    return logits, scores


@pytest.mark.parametrize("V,live,seed", MANY)
def test_many_picks(gpu, V, live, seed):
    """64 picks of 64 beams: few beams that go on (the rest wait at -inf), rows with few tokens allowed, a row that has none."""
    from tensorpack_amd.sampling import beam_select
    logits, scores = _many(V, live, seed)
    for n in (17, 25, 64):
        want = _want(logits, scores, n)
        _check(beam_select(logits.to(gpu), scores.to(gpu), n=n), want)


@pytest.mark.parametrize("V,W", [(40, 2), (3000, 3), (600000, 16)])
def test_equal_scores_in_the_order_of_places(gpu, V, W):
    """Rows of one value (more equal ones than any list holds), and equal beams: the lowest places come first."""
    import torch
    from tensorpack_amd.sampling import beam_select
    for dtype in (torch.float32, torch.bfloat16):
        logits, scores = torch.zeros((2, W, V), dtype=dtype, device=gpu), torch.zeros((2, W), device=gpu)
        n = 20
        s, t, p = beam_select(logits, scores, n=n)
        flat = np.arange(n)
        assert t.tolist() == [(flat % V).tolist()] * 2 and p.tolist() == [(flat // V).tolist(), (flat // V + W).tolist()]
        assert float((s + math.log(V)).abs().max()) <= LOG_ERROR + 2.0 ** -24 * 16
        logits[:, 1, V // 2:] = 1.0
        logits[:, 1, V - 1] = 2.0
        s, t, p = beam_select(logits, torch.tensor([[0.0, 30.0] + [0.0] * (W - 2)] * 2, device=gpu), n=min(n, V // 2))
        assert t[0].tolist() == [V - 1] + list(range(V // 2, V // 2 + t.shape[1] - 1)) and set(p[1].tolist()) == {W + 1}


def test_masked_tokens_and_bad_rows(gpu):
    """-inf logits are no candidates; a beam with a NaN or +inf, or with nothing but -inf, has none; the others are not touched."""
    import torch
    from tensorpack_amd.sampling import beam_select
    g = torch.Generator().manual_seed(3)
    for V in (600, 9000):
        logits = torch.randn((1, 6, V), generator=g).to(gpu)
        logits[0, 0, 5:] = -math.inf
        logits[0, 1, V // 3] = math.nan
        logits[0, 2, V - 1] = math.inf
        logits[0, 3] = -math.inf
        logits[0, 4, ::2] = -math.inf
        scores = torch.tensor([[-1.0, 0.0, 0.0, 0.0, -2.0, math.nan]], device=gpu)
        s, t, p = beam_select(logits, scores, n=12)
        want = _want(logits[:, [0, 4]], scores[:, [0, 4]], 12)[0]
        assert t[0].tolist() == [r[1] for r in want] and p[0].tolist() == [(0, 4)[r[2]] for r in want]
        assert torch.isfinite(s).all()
        s, t, p = beam_select(logits[:, 1:4], scores[:, 1:4])
        assert t.tolist() == [[-1] * 3] and p.tolist() == [[0, 1, 2]] and (s == -math.inf).all()
        first = beam_select(logits[:, :1], scores[:, :1], n=8)
        assert first[1][0, 5:].tolist() == [-1] * 3 and sorted(first[1][0, :5].tolist()) == list(range(5))


def test_close_logits_of_far_scores(gpu):
    """Differences that fp32 scores would lose: logits apart by their last bit under a score of -1e6."""
    import torch
    from tensorpack_amd.sampling import beam_select
    logits = torch.full((1, 1, 2000), 1.0, device=gpu)
    for i, at in enumerate((1500, 3, 777)):
        logits[0, 0, at] = 1.0 + (3 - i) * 2.0 ** -23
    s, t, p = beam_select(logits, torch.full((1, 1), -1e6, device=gpu), n=4)
    assert t[0].tolist() == [1500, 3, 777, 0]


def test_views(gpu):
    import torch
    from tensorpack_amd.sampling import beam_select
    g = torch.Generator().manual_seed(4)
    base = torch.randn((3, 2, 5, 1003), generator=g).bfloat16().to(gpu)
    scores = torch.rand((3, 5), generator=g).to(gpu)
    for x in (base[:, 1], base[:, 0, :, 1:1000], base.transpose(1, 3)[:, :, :, 0].transpose(1, 2)[..., :900], base[:1, 0].expand(3, 5, 1003)):
        got, want = beam_select(x, scores), beam_select(x.contiguous(), scores)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = beam_select(base[:, 1], torch.stack([scores, scores], -1)[..., 0], done=torch.zeros((5, 3), dtype=torch.bool, device=gpu).t())
    assert all(torch.equal(a, b) for a, b in zip(got, beam_select(base[:, 1], scores)))


def test_rows_far_apart(gpu):
    """Rows 2 GiB apart: offsets pass 32 bits."""
    import torch
    from tensorpack_amd.sampling import beam_select
    buf = torch.empty((3 << 30) + 4096, dtype=torch.bfloat16, device=gpu)
    far = buf.as_strided((2, 2, 2003), (2 << 30, 1 << 30, 1), 5)
    near = torch.randn((2, 2, 2003), generator=torch.Generator().manual_seed(6)).bfloat16().to(gpu)
    far.copy_(near)
    scores = torch.tensor([[-1.0, -1.5], [-3.0, -2.0]], device=gpu)
    assert all(torch.equal(a, b) for a, b in zip(beam_select(far, scores), beam_select(near, scores)))


def test_capture_and_stream(gpu):
    import torch
    from tensorpack_amd.sampling import beam_select
    logits, scores = torch.randn((2, 4, 9000), device=gpu), torch.zeros((2, 4), device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = beam_select(logits, scores)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, beam_select(logits, scores)))
    graphs = []
    for _ in range(2):                                           # each with its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = beam_select(logits, scores)
        graphs.append((g, out))
    for step in range(4):
        logits.copy_(torch.randn(logits.shape, generator=torch.Generator().manual_seed(step)))
        for g, _ in graphs:
            g.replay()
        want = beam_select(logits, scores)
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_search_finds_the_best_sentences(gpu):
    """A step of beam search as a program runs it, on a cache and without: the beams after each step are the best continuations of
    the kept ones, and each beam's cache holds its own tokens."""
    import torch
    from tensorpack_amd.cache import PagedCache
    from tensorpack_amd.sampling import beam_select
    V, W, B, steps = 40, 4, 2, 20
    table = torch.log_softmax(2 * torch.randn((B, V, V), generator=torch.Generator().manual_seed(6)), -1).to(gpu)    # next given last
    cache = PagedCache(80, 1, 1, 8, max_seqs=B * W, max_pages=4, device=gpu)
    seqs, one, cu = _ints(list(range(B * W)), gpu), _ints([1] * (B * W), gpu), _ints(list(range(B * W + 1)), gpu)
    last = torch.zeros((B, W), dtype=torch.long, device=gpu)
    scores = torch.tensor([[0.0] + [-math.inf] * (W - 1)] * B, device=gpu)
    texts = [[[0] for _ in range(W)] for _ in range(B)]
    for step in range(steps):
        cache.extend(seqs, one)
        x = last.flatten()[:, None, None].expand(B * W, 1, 8).to(torch.bfloat16).contiguous()
        cache.append(0, x, x, seqs, cu)
        logits = table[torch.arange(B, device=gpu)[:, None], last] + 5.0                       # any shift of the logits
        scores, tokens, parents = beam_select(logits, scores)
        cache.reorder(seqs, parents.view(-1))
        last = tokens.long()
        texts = [[texts[b][p % W] + [t] for p, t in zip(parents[b].tolist(), tokens[b].tolist())] for b in range(B)]
    cache.check()
    for b in range(B):
        for w in range(W):
            text = texts[b][w]
            assert abs(sum(float(table[b, x, y]) for x, y in zip(text, text[1:])) - float(scores[b, w])) < 20 * (LOG_ERROR + 60 * 2.0 ** -24)
            s = b * W + w
            held = cache.pool[cache.table[s, :2].long(), 0, 0, 0, :, 0].flatten()[:steps]
            assert held.int().tolist() == text[:steps]
        assert len(set(map(tuple, texts[b]))) == W


def test_refusals(gpu):
    import torch
    from tensorpack_amd.sampling import beam_select
    x, s = torch.zeros((2, 3, 10), device=gpu), torch.zeros((2, 3), device=gpu)
    for a, b, kw in ((x[0], s, {}), (x, s[:1], {}), (x, s.double(), {}), (x.double(), s, {}), (x, s, {"n": 0}), (x, s, {"n": 65}), (x[:, :, :0], s, {}),
                     (x, s.cpu(), {}), (x, s, {"done": s}), (x, s, {"done": (s[:1] > 0)}), (x, s, {"done": (s > 0).cpu()}), (x, s, {"pad": 1 << 31}),
                     (x[:, :0], s[:, :0], {}), (torch.zeros((1, 65, 4), device=gpu), torch.zeros((1, 65), device=gpu), {})):
        with pytest.raises(ValueError):
            beam_select(a, b, **kw)
    assert [t.shape for t in beam_select(x[:0], s[:0])] == [(0, 3)] * 3
