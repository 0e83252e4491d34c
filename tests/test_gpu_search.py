"""Rotary positions, the 8-bit cache, attention over it and the beam step together, as examples/search_beams.py runs them over
packed layers."""

import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("search_beams", os.path.join(ROOT, "examples", "search_beams.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def decoder(example, gpu):
    return example.RotaryDecoder(gpu, width=128, heads=4, kv_heads=2, head_dim=32, inner=128, vocab=128)


PROMPTS = [np.random.RandomState(3).randint(0, 128, 50), np.random.RandomState(4).randint(0, 128, 33)]


def test_scores_are_those_of_the_texts(example, decoder, gpu):
    """Each beam's score is the sum of its tokens' log probabilities when its text is fed to the decoder alone, one token after
    another. The two differ by roundings to 16 and 8 bits of inputs that differ in their last bits (the products of 8 rows and of
    one are different kernels): a few 2^-8 of the logits' root mean square each (2 to 4 here), at most 5 % of it, twice that in a log
    probability, on 10 tokens at most 4. Histories that were mixed up change logits by all of their size, at every token."""
    import torch
    found = example.search(decoder, PROMPTS, beams=4, tokens=10)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    worst = 0.0
    for b, best in enumerate(found):
        assert all(x[0] >= y[0] for x, y in zip(best, best[1:])) and len({tuple(t) for _, t in best}) == 4
        for score, text in best:
            cache = decoder.cache(1)
            logits = decoder.prompts(torch.as_tensor(PROMPTS[b], device=gpu), ints([0, len(PROMPTS[b])]), cache, ints([0]))
            total = 0.0
            for t in text:
                total += float(torch.log_softmax(logits[0].double(), -1)[t])
                logits = decoder.step(torch.tensor([t], device=gpu), cache, ints([0]))
            worst = max(worst, abs(total - score))
    assert worst < 4.0 * 0.1 * 10, worst


def test_a_wider_search_finds_no_worse(example, decoder, gpu):
    """One beam is the greedy text; the same call twice gives the same texts."""
    one = example.search(decoder, PROMPTS, beams=1, tokens=8)
    assert one == example.search(decoder, PROMPTS, beams=1, tokens=8)
    six = example.search(decoder, PROMPTS, beams=6, tokens=8)
    assert six == example.search(decoder, PROMPTS, beams=6, tokens=8)
    assert all(len(t) == 8 for best in six for _, t in best)


def test_ended_beams_stay(example, decoder, gpu):
    """With an end token that comes often, beams end at different steps and stay as they are."""
    free = example.search(decoder, PROMPTS, beams=4, tokens=6)
    end = free[0][0][1][1]
    out = example.search(decoder, PROMPTS, beams=4, tokens=12, end=end)
    ended = [t for best in out for _, t in best if end in t]
    assert ended and all(t.index(end) == len(t) - 1 for t in ended)
    assert all(np.isfinite(s) for best in out for s, _ in best)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_a_captured_step(gpu, dtype):
    """A step of all calls (a token more of each beam, positions, append, attention with the prompts shared, selection, reordering)
    captured once and replayed, against eager steps on a cache of its own, bit by bit; the eager ones run between the replays."""
    import torch
    from tensorpack_amd.attention import cached_attention
    from tensorpack_amd.cache import QuantizedCache
    from tensorpack_amd.rotary import Rotary, apply_rotary
    from tensorpack_amd.sampling import beam_select
    dtype = getattr(torch, dtype)
    n, beams, heads, kv, dim, vocab = 3, 4, 6, 2, 40, 1500
    rows = n * beams
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    g = torch.Generator().manual_seed(5)
    rand = lambda *shape: torch.randn(shape, generator=g).to(gpu).to(dtype)
    lens = [37, 1, 64]
    rotary = Rotary(32, interleaved=True, device=gpu)
    roots, seqs, cu, ones = ints(range(n)), ints(range(n, n + rows)), ints(range(rows + 1)), ints([1] * rows)
    groups, prefix, starts = ints(range(0, rows + 1, beams)), ints(lens), ints(np.concatenate([[0], np.cumsum(lens)]).tolist())
    first = rand(2, sum(lens), kv, dim)

    class Side:
        def __init__(self):
            self.cache = QuantizedCache(200, 1, kv, dim, max_seqs=n + rows, max_pages=8, dtype=dtype, device=gpu)
            self.cache.extend(roots, prefix)
            self.cache.append(0, first[0], first[1], roots, starts)
            self.cache.fork(roots.repeat_interleave(beams), seqs)
            self.q, self.k, self.v = (torch.empty((rows, h, dim), dtype=dtype, device=gpu) for h in (heads, kv, kv))
            self.logits = torch.empty((n, beams, vocab), device=gpu)
            self.scores, self.done = torch.zeros((n, beams), device=gpu), torch.zeros((n, beams), dtype=torch.bool, device=gpu)

        def take(self, inputs):
            for a, b in zip((self.q, self.k, self.v, self.logits), inputs):
                a.copy_(b)

        def step(self):
            c = self.cache
            c.extend(seqs, ones)
            q, k = apply_rotary(rotary, self.q, self.k, c.lens[seqs.long()] - 1)
            c.append(0, k, self.v, seqs, cu)
            self.o = cached_attention(q[:, None], c, 0, seqs, groups=groups, prefix_lens=prefix)
            scores, self.tokens, self.parents = beam_select(self.logits, self.scores, done=self.done, pad=9)
            self.scores.copy_(scores)
            self.done.copy_(self.done.gather(1, self.parents.long() % beams) | (self.tokens % 50 == 3))
            c.reorder(seqs, self.parents.view(-1))

    eager, captured = Side(), Side()
    inputs = lambda: (rand(rows, heads, dim), rand(rows, kv, dim), rand(rows, kv, dim) * 3, rand(n, beams, vocab).float() * 4)
    x = inputs()
    for side in (eager, captured):
        side.take(x)
        side.step()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        captured.step()
    for i in range(30):
        x = inputs()
        captured.take(x)
        graph.replay()
        if i % 3 == 0:
            torch.cuda.synchronize()
        eager.take(x)
        eager.step()
        assert torch.isfinite(eager.o).all() and bool(eager.o.abs().sum(-1).min() > 0)
        for name in ("o", "tokens", "parents", "scores", "done"):
            assert torch.equal(getattr(eager, name), getattr(captured, name)), (i, name)
        assert torch.equal(eager.cache.lens, captured.cache.lens) and torch.equal(eager.cache.table, captured.cache.table)
    assert int(eager.cache.lens[int(seqs[0])]) == lens[0] + 31
    for side in (eager, captured):
        side.cache.check()
        side.cache.free(torch.cat([roots, seqs]))
        assert side.cache.free_pages == 200
