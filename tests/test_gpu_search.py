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
