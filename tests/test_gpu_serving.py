"""The serving operators together, as examples/sample_with_drafts.py runs them over packed layers."""

import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("sample_with_drafts", os.path.join(ROOT, "examples", "sample_with_drafts.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def decoder(example, gpu):
    return example.Decoder(gpu, width=128, heads=4, kv_heads=2, head_dim=32, inner=128, vocab=128)


def test_cached_logits_are_the_prompt_s(example, decoder, gpu):
    """The same tokens through the cache (prompt, fork, then 5 and 3 at a time, a shared prefix) and as one prompt: both
    round Q, K, V and the attention's result to bf16 from inputs that differ by such roundings (2^-8 each, two
    layers of residual sums), so logits of size 2 to 8 agree to a few 2^-8 of their root mean square; 5 %."""
    import torch
    rng = np.random.RandomState(3)
    head, tails = rng.randint(0, 128, 50), rng.randint(0, 128, (3, 8))
    cache = decoder.cache(answers=3)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    decoder.prompt(torch.as_tensor(head, device=gpu), cache, ints([0]))
    seqs = ints([1, 2, 3])
    cache.fork(ints([0, 0, 0]), seqs)
    t = torch.as_tensor(tails, device=gpu)
    got = torch.cat([decoder.extend(t[:, :5], cache, seqs, ints([0, 3]), ints([50])),
                     decoder.extend(t[:, 5:], cache, seqs, None, None)], 1)
    cache.check()
    for i in range(3):
        want = decoder.prompt(torch.as_tensor(np.concatenate([head, tails[i]]), device=gpu))[50:]
        err = float((got[i] - want).square().mean().sqrt() / want.square().mean().sqrt())
        assert err < 0.05, err


def test_sampling(example, decoder, gpu):
    prompt = np.random.RandomState(1).randint(0, 128, 40).tolist()
    out, rounds, kept = example.sample(decoder, prompt, answers=3, tokens=24, drafts=3, seed=5)
    assert all(len(x) >= 24 and min(x) >= 0 and max(x) < 128 for x in out)
    assert 0 < kept <= rounds * 9 and rounds < 24
    assert out == example.sample(decoder, prompt, answers=3, tokens=24, drafts=3, seed=5)[0]        # the same numbers, the same answers


def test_sampling_distribution(example, decoder, gpu):
    """The second token of an answer, drafted and verified, against the decoder's own probabilities given the first: chi-square
    over the most frequent first token's answers, bins of at least 5 expected."""
    import torch
    prompt = [5, 17, 99]
    pairs = []
    for seed in range(60):
        out, _, _ = example.sample(decoder, prompt, answers=16, tokens=2, drafts=1, seed=seed)
        pairs += [tuple(x[:2]) for x in out]
    first = max(set(p[0] for p in pairs), key=[p[0] for p in pairs].count)
    second = np.bincount([b for a, b in pairs if a == first], minlength=128)
    p = torch.softmax(decoder.prompt(torch.tensor(prompt + [first], device=gpu))[-1].double(), -1).cpu().numpy()
    n = second.sum()
    order = np.argsort(-p)
    bins, rest = [], [0.0, 0]
    for i in order:
        if n * p[i] >= 5:
            bins.append((n * p[i], second[i]))
        else:
            rest = [rest[0] + n * p[i], rest[1] + second[i]]
    if rest[0] > 0:
        bins.append(tuple(rest))
    chi = sum((o - e) ** 2 / e for e, o in bins)
    assert len(bins) > 2 and chi < len(bins) - 1 + 6 * (2 * (len(bins) - 1)) ** 0.5, (chi, len(bins))
