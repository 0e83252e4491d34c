"""Beam search over a small decoder of packed layers with rotary positions and an 8-bit cache.

    python examples/search_beams.py [--prompts 2] [--beams 4] [--tokens 32]

The decoder is that of `sample_with_drafts.py` (random weights, packed layers) with positions; each step runs

- `apply_rotary` on q and k, at the places that the tokens have in their sequences;
- `append` into a `QuantizedCache`, which holds K and V in 8 bits, and `cached_attention` over it; the beams of a prompt are forks of
  it, whose pages are read once for all of them (`groups`, `prefix_lens`);
- `beam_select`: the best continuations of each prompt's beams, with the beams that they come from, and `reorder`, which gives
  each beam the cache of the one that it goes on from. `extend` copies a page when a beam writes into one that others hold too.
A beam that has written the end token stands as it is from then on.
"""

import argparse
import math
import os
import sys
import time

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "examples")):
    if p not in sys.path:
        sys.path.insert(0, p)

from sample_with_drafts import Decoder, _norm                                # noqa: E402
from tensorpack_amd.attention import cached_attention, prompt_attention      # noqa: E402
from tensorpack_amd.cache import QuantizedCache                              # noqa: E402
from tensorpack_amd.rotary import Rotary, apply_rotary                       # noqa: E402
from tensorpack_amd.sampling import beam_select                              # noqa: E402


class RotaryDecoder(Decoder):
    """Decoder with rotary positions over an 8-bit cache; its context is stretched fourfold from 256 tokens."""

    def __init__(self, device, **kw):
        super().__init__(device, **kw)
        self.rotary = Rotary(self.head_dim, factor=4.0, original=256, device=device)

    def cache(self, sequences, pages=256):
        return QuantizedCache(pages, len(self.layers), self.kv_heads, self.head_dim, max_seqs=sequences, max_pages=64, device=self.device)

    def _attended(self, q, k, positions):
        return apply_rotary(self.rotary, q, k.contiguous(), positions)

    def prompts(self, tokens, cu, cache, seqs):
        """Logits after the last token of each prompt, packed one after another at cu; K and V are kept as sequences `seqs`."""
        ends = cu[1:].long()
        lens = cu[1:] - cu[:-1]
        cache.extend(seqs, lens)
        positions = torch.arange(tokens.shape[0], dtype=torch.int32, device=self.device)
        positions -= torch.repeat_interleave(cu[:-1], lens.long(), output_size=tokens.shape[0])
        x = self.embedding[tokens]
        for i, p in enumerate(self.layers):
            def attend(q, k, v):
                q, k = self._attended(q, k.bfloat16(), positions)
                cache.append(i, k, v.bfloat16(), seqs, cu)
                return prompt_attention(q, k, v.bfloat16(), cu)
            x = self._layer(p, x, attend)
        return self.head(_norm(x[ends - 1]), compute="fp32")

    def step(self, tokens, cache, seqs, groups=None, prefix=None):
        """Logits (sequences, vocab) after one more token of each sequence."""
        n = tokens.shape[0]
        cu = torch.arange(n + 1, dtype=torch.int32, device=self.device)
        cache.extend(seqs, torch.ones(n, dtype=torch.int32, device=self.device))
        positions = cache.lens[seqs.long()] - 1
        x = self.embedding[tokens]
        for i, p in enumerate(self.layers):
            def attend(q, k, v):
                q, k = self._attended(q, k.bfloat16(), positions)
                cache.append(i, k, v.bfloat16(), seqs, cu)
                return cached_attention(q[:, None], cache, i, seqs, groups=groups, prefix_lens=prefix)[:, 0]
            x = self._layer(p, x, attend)
        return self.head(_norm(x), compute="fp32")


def search(decoder, prompts, beams=4, tokens=32, end=None):
    """The best `beams` continuations of each prompt, of up to `tokens` tokens: [[(score, tokens)]], best first."""
    dev, n = decoder.device, len(prompts)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    cache = decoder.cache(n + n * beams)
    roots, seqs = ints(range(n)), ints(range(n, n + n * beams))
    cu = ints(np.concatenate([[0], np.cumsum([len(p) for p in prompts])]).tolist())
    logits = decoder.prompts(torch.as_tensor(np.concatenate(prompts), device=dev), cu, cache, roots)
    cache.fork(roots.repeat_interleave(beams), seqs)
    groups, prefix = ints(range(0, n * beams + 1, beams)), cu[1:] - cu[:-1]
    # the first step: every beam is the prompt, so only one of them may go on
    logits = logits[:, None].expand(-1, beams, -1)
    scores = torch.full((n, beams), -math.inf, device=dev)
    scores[:, 0] = 0.0
    done = torch.zeros((n, beams), dtype=torch.bool, device=dev)
    texts = torch.zeros((n * beams, 0), dtype=torch.int32, device=dev)
    for t in range(tokens):
        scores, chosen, parents = beam_select(logits, scores, done=done, pad=end or 0)
        rows = parents.view(-1)
        cache.reorder(seqs, rows)
        texts = torch.cat([texts[rows.long()], chosen.view(-1, 1)], 1)
        if end is not None:
            done = done.view(-1)[rows.long()].view(n, beams) | (chosen == end)
        if t + 1 < tokens:
            logits = decoder.step(chosen.view(-1).clamp(min=0).long(), cache, seqs, groups, prefix).view(n, beams, -1)
    cache.check()
    cache.free(torch.cat([roots, seqs]))
    assert cache.free_pages == cache.n_pages
    out = []
    for b, row in enumerate(texts.view(n, beams, -1).tolist()):
        cut = [t[:t.index(end) + 1] if end in t else t for t in row]
        out.append(list(zip(scores[b].tolist(), cut)))
    return out


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompts", type=int, default=2)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=32)
    a = ap.parse_args(argv)
    decoder = RotaryDecoder(torch.device("cuda", torch.cuda.current_device()))
    rng = np.random.RandomState(1)
    prompts = [rng.randint(0, decoder.vocab, size=60 + 17 * i) for i in range(a.prompts)]
    search(decoder, prompts, a.beams, 2)                                 # packs the weights, loads the kernels
    t = time.perf_counter()
    out = search(decoder, prompts, a.beams, a.tokens, end=7)
    dt = time.perf_counter() - t
    for b, best in enumerate(out):
        print(f"prompt {b}: best {best[0][0]:.3f} ({len(best[0][1])} tokens), last {best[-1][0]:.3f}")
    print(f"{a.tokens} steps of {a.prompts} x {a.beams} beams, {1e3 * dt / a.tokens:.2f} ms a step")


if __name__ == "__main__":
    main()
