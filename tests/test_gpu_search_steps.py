"""examples/search_beams.py step by step: what beam_select was given and gave at each step, against the definition in 64 bits, and the texts that
come out of it; one beam against a greedy loop over the same decoder.

Bound of a step: of 128 terms a log sum is off by less than 10 * 2^-24 for its sums, 3 * 2^-24 for the exponentials and 2.3 * 2^-24 times their distance
from the maximum by their share, at most 2.9 (x d / (1 + x) of x = 128 exp(-d)): 20 * 2^-24 together; a score is rounded once, 2^-24 of it."""

import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROMPTS = [np.random.RandomState(3).randint(0, 128, 50), np.random.RandomState(4).randint(0, 128, 33)]


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("search_beams", os.path.join(ROOT, "examples", "search_beams.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def decoder(example, gpu):
    return example.RotaryDecoder(gpu, width=128, heads=4, kv_heads=2, head_dim=32, inner=128, vocab=128)


def _recorded(example, monkeypatch):
    steps = []

    def select(logits, scores, *, done, pad):
        out = beam_select(logits, scores, done=done, pad=pad)
        steps.append((logits.double().cpu().numpy(), scores.cpu().numpy(), done.cpu().numpy(), pad, *(x.cpu().numpy() for x in out)))
        return out

    from tensorpack_amd.sampling import beam_select
    monkeypatch.setattr(example, "beam_select", select)
    return steps


def _bound(score):
    return 20 * 2.0 ** -24 + 2.0 ** -24 * abs(score)


@pytest.mark.parametrize("beams,ends", [(4, False), (6, False), (5, True), (1, False)])
def test_every_step_and_the_texts(example, decoder, gpu, monkeypatch, beams, ends):
    end = example.search(decoder, PROMPTS, beams=beams, tokens=3)[0][0][1][1] if ends else None         # a token that comes
    steps = _recorded(example, monkeypatch)
    found = example.search(decoder, PROMPTS, beams=beams, tokens=10, end=end)
    assert len(steps) == 10
    n = len(PROMPTS)
    texts, sums, over = [[[]] * beams for _ in range(n)], np.zeros((n, beams)), np.zeros((n, beams), bool)
    for t, (logits, scores, done, pad, best, tokens, parents) in enumerate(steps):
        top = logits.max(-1, keepdims=True)
        logp = logits - top - np.log(np.exp(logits - top).sum(-1, keepdims=True))
        assert np.array_equal(done, over)
        if t:
            assert np.array_equal(scores, steps[t - 1][4])           # as they came out
        new_texts, new_sums, new_over = [], np.zeros((n, beams)), np.zeros((n, beams), bool)
        for b in range(n):
            all_ = {}
            for w in range(beams):
                if done[b, w]:
                    all_[w, pad] = float(scores[b, w])
                elif scores[b, w] > -np.inf:
                    all_.update({(w, v): float(scores[b, w]) + logp[b, w, v] for v in range(logits.shape[2])})
            got = [(int(parents[b, i]) - b * beams, int(tokens[b, i])) for i in range(beams)]
            assert len(set(got)) == beams and all(abs(all_[g] - s) <= _bound(s) for g, s in zip(got, best[b]))
            assert (np.diff(best[b]) <= 0).all()
            left = [s for g, s in all_.items() if g not in got]
            assert max(left) <= best[b].min() + 2 * _bound(best[b].min())
            new_texts.append([texts[b][w] + [v] for w, v in got])
            for i, (w, v) in enumerate(got):
                new_sums[b, i] = sums[b, w] + (0.0 if done[b, w] else logp[b, w, v])
                new_over[b, i] = done[b, w] or (end is not None and v == end)
        texts, sums, over = new_texts, new_sums, new_over
    if end is not None:
        assert over.any()
    for b in range(n):
        cut = [x[:x.index(end) + 1] if end in x else x for x in texts[b]]
        assert [list(x) for _, x in found[b]] == cut
        assert all(abs(s - y) <= 10 * _bound(y) for (s, _), y in zip(found[b], sums[b]))


def test_one_beam_is_the_greedy_text(example, decoder, gpu):
    """The same calls of the decoder with the largest logit taken each time."""
    import torch
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    n, count = len(PROMPTS), 12
    found = example.search(decoder, PROMPTS, beams=1, tokens=count)
    cache = decoder.cache(2 * n)
    roots, seqs, cu = ints(range(n)), ints(range(n, 2 * n)), ints(np.concatenate([[0], np.cumsum([len(p) for p in PROMPTS])]).tolist())
    logits = decoder.prompts(torch.as_tensor(np.concatenate(PROMPTS), device=gpu), cu, cache, roots)
    cache.fork(roots, seqs)
    total, texts = np.zeros(n), [[] for _ in range(n)]
    for t in range(count):
        logp = torch.log_softmax(logits.double(), -1).cpu().numpy()
        token = logits.argmax(-1)
        for b, v in enumerate(token.tolist()):
            texts[b].append(v)
            total[b] += logp[b, v]
        if t + 1 < count:
            logits = decoder.step(token, cache, seqs, ints(range(n + 1)), cu[1:] - cu[:-1])
    assert [best[0][1] for best in found] == texts
    assert all(abs(best[0][0] - s) <= count * _bound(s) for best, s in zip(found, total))
