"""Sampling several answers to one prompt from a small decoder of packed layers, with drafted tokens.

    python examples/sample_with_drafts.py [--answers 4] [--tokens 64] [--drafts 4]

The decoder (random weights) is built from this package's parts: `LinearMTCGroup` for the q/k/v and gate/up products,
`LinearMTC` for the others, and between them the serving operators:

- the prompt goes through `prompt_attention`; its K and V into a `PagedCache` (`extend`, `append`);
- the answers are forks of the prompt: they share its pages (`fork`; `extend` copies the partly filled last one), and
  `cached_attention` reads them once for all answers (`groups`, `prefix_lens`);
- drafts come from the first layer and the head alone. That layer's K and V are the decoder's own, so the draft uses the
  same cache and `truncate` takes its tokens back; then all layers score the drafts in one pass of
  drafts + 1 rows per answer (at up to 16 rows the packed products read their weights once, as for one row);
- `verify_drafts` keeps a run of drafts and draws the next token, so that the answers are distributed as the
  decoder's own; `truncate` drops the K and V of the rejected ones;
- at the end the answers are freed and the cache is compacted.
"""

import argparse
import os
import sys
import time

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from tensorpack_amd.attention import cached_attention, prompt_attention      # noqa: E402
from tensorpack_amd.cache import PagedCache                                  # noqa: E402
from tensorpack_amd.nn import LinearMTC, LinearMTCGroup                      # noqa: E402
from tensorpack_amd.sampling import verify_drafts                            # noqa: E402


def _norm(x):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)


class Decoder:
    """layers of attention (heads of head_dim over kv_heads) and a gated product, normalised inputs, no positions."""

    def __init__(self, device, *, layers=2, width=256, heads=4, kv_heads=2, head_dim=64, inner=512, vocab=512, bits=4.25, seed=0):
        self.device, self.heads, self.kv_heads, self.head_dim, self.vocab = device, heads, kv_heads, head_dim, vocab
        rng = np.random.RandomState(seed)

        def linear(n_in, n_out, gain=1.0):
            w = (rng.randn(n_in, n_out) * gain / np.sqrt(n_in)).astype(np.float32)
            return LinearMTC(n_in, n_out, bits, weight=w, permuted=False)
        kv = kv_heads * head_dim
        self.layers = [{"qkv": LinearMTCGroup([linear(width, heads * head_dim, 1.5), linear(width, kv), linear(width, kv)]),
                        "o": linear(heads * head_dim, width), "gate_up": LinearMTCGroup([linear(width, inner), linear(width, inner)]),
                        "down": linear(inner, width)} for _ in range(layers)]
        self.head = linear(width, vocab, 2.0)
        g = torch.Generator().manual_seed(seed)
        self.embedding = torch.randn((vocab, width), generator=g).to(device)

    def cache(self, pages=256, answers=16):
        return PagedCache(pages, len(self.layers), self.kv_heads, self.head_dim, max_seqs=answers + 1, max_pages=64, device=self.device)

    def _layer(self, p, x, attend):
        q, k, v = p["qkv"](_norm(x), compute="fp32")
        q, k, v = (t.unflatten(-1, (-1, self.head_dim)) for t in (q, k, v))
        x = x + p["o"](attend(q.bfloat16(), k, v).flatten(-2).float(), compute="fp32")
        gate, up = p["gate_up"](_norm(x), compute="fp32")
        return x + p["down"](torch.nn.functional.silu(gate) * up, compute="fp32")

    def prompt(self, tokens, cache=None, seq=None):
        """Logits after every token of one prompt; with a cache its K and V are kept there as sequence `seq`."""
        n = tokens.shape[0]
        cu = torch.tensor([0, n], dtype=torch.int32, device=self.device)
        if cache is not None:
            cache.extend(seq, torch.tensor([n], dtype=torch.int32, device=self.device))
        x = self.embedding[tokens]
        for i, p in enumerate(self.layers):
            def attend(q, k, v):
                if cache is not None:
                    cache.append(i, k, v, seq, cu)                       # fp32, rounded on the way
                return prompt_attention(q, k.bfloat16(), v.bfloat16(), cu)
            x = self._layer(p, x, attend)
        return self.head(_norm(x), compute="fp32")

    def extend(self, tokens, cache, seqs, groups, prefix, layers=None):
        """Logits (sequences, tokens, vocab) after each new token; tokens (sequences, count)."""
        b, t = tokens.shape
        cu = torch.arange(b + 1, dtype=torch.int32, device=self.device) * t
        cache.extend(seqs, torch.full((b,), t, dtype=torch.int32, device=self.device))
        x = self.embedding[tokens.flatten()]
        for i, p in enumerate(self.layers[:layers]):
            def attend(q, k, v):
                cache.append(i, k, v, seqs, cu)
                out = cached_attention(q.unflatten(0, (b, t)), cache, i, seqs, groups=groups, prefix_lens=prefix)
                return out.flatten(0, 1)
            x = self._layer(p, x, attend)
        return self.head(_norm(x), compute="fp32").unflatten(0, (b, t))


def _race(shape, device, gen):
    return 1.0 / torch.empty(shape, device=device).exponential_(generator=gen).clamp_min(1e-20)


def sample(decoder, prompt, answers=4, tokens=64, drafts=4, seed=0):
    """(answers as lists of tokens, rounds, drafts accepted): `tokens` or a few more tokens per answer."""
    dev = decoder.device
    gen = torch.Generator(device=dev).manual_seed(seed)
    cache = decoder.cache(answers=answers)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    root, seqs = ints([0]), ints(range(1, answers + 1))
    prompt = torch.as_tensor(prompt, device=dev)
    p = torch.softmax(decoder.prompt(prompt, cache, root)[-1:], -1)
    cache.fork(root.repeat(answers), seqs)
    groups, prefix = ints([0, answers]), ints([prompt.shape[0]])
    last = (p * _race((answers, decoder.vocab), dev, gen)).argmax(-1, keepdim=True)      # each answer's first token
    out = [[int(x)] for x in last[:, 0].tolist()]
    rounds = kept = 0
    while min(len(x) for x in out) < tokens:
        before = cache.lens[seqs.long()]
        drafted, q = [last], []
        for _ in range(drafts):
            q.append(torch.softmax(decoder.extend(drafted[-1], cache, seqs, groups, prefix, layers=1)[:, 0], -1))
            drafted.append((q[-1] * _race((answers, decoder.vocab), dev, gen)).argmax(-1, keepdim=True))
        cache.truncate(seqs, before)                                     # the drafts' K and V come again with all layers
        new = torch.cat(drafted, 1)
        p = torch.softmax(decoder.extend(new, cache, seqs, groups, prefix), -1)
        got, count = verify_drafts(new[:, 1:].contiguous(), p, torch.stack(q, 1), torch.rand((answers, drafts), device=dev, generator=gen),
                                   _race((answers, decoder.vocab), dev, gen))
        cache.truncate(seqs, before + 1 + count)
        last = got.gather(1, count[:, None].long())
        for x, row, n in zip(out, got.tolist(), count.tolist()):
            x += row[:n + 1]
            kept += n
        rounds += 1
    cache.check()
    cache.free(torch.cat([root, seqs]))
    cache.compact()
    assert cache.free_pages == cache.n_pages
    return out, rounds, kept


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--answers", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--drafts", type=int, default=4)
    a = ap.parse_args(argv)
    decoder = Decoder(torch.device("cuda", torch.cuda.current_device()))
    prompt = list(np.random.RandomState(1).randint(0, decoder.vocab, size=100))
    sample(decoder, prompt, a.answers, 4, a.drafts)                      # packs the weights, loads the kernels
    t = time.perf_counter()
    out, rounds, kept = sample(decoder, prompt, a.answers, a.tokens, a.drafts)
    dt = time.perf_counter() - t
    n = sum(len(x) for x in out)
    print(f"{n} tokens in {rounds} rounds, {kept} of {rounds * a.drafts * a.answers} drafts accepted, {1e3 * dt:.1f} ms")


if __name__ == "__main__":
    main()
