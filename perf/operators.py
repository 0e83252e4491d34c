"""Workloads of the serving operators around the packed linear layers, for timing and for comparing results.

  prompt  prompt_attention: whole prompts (or a chunk of new tokens on older ones), packed one after another
  cached  cached_attention: the last few tokens of each sequence over a paged cache, with or without groups
          of sequences that share a long prefix
  pages   PagedCache: sampled continuations forked from prompts, extended (copy on write) and appended to;
          a fragmented cache compacted
  verify  verify_drafts: drafted tokens against the target's probabilities

With `own` false, `run` computes them in plain torch operations in 32 bits, rounded once at the end; with `own`
true it makes the calls a program makes. Both get the same tensors from `prepare`.

Case fields
  op        prompt | cached | pages | verify
  dtype     bf16 | fp16 | fp32: type of q, k, v, the cache or the probabilities
  heads, kv_heads, dim, page, layers     shapes of attention and cache
  n         sequences; longest: tokens (keys) of the longest; ragged: the others are shorter, some are empty
  pattern   seed of what belongs to the case, not to the inputs: lengths, places of pages
  causal, new, fused   (prompt) new: queries per sequence on longer keys (0: all); fused: q, k, v are views of one tensor
  tokens, prefix, members   (cached) queries per sequence, tokens of a shared prefix, sequences per group
  kind, ways, pages    (pages) fork | compact, continuations per prompt, pages of the pool
  drafts, vocab, close (verify) drafted tokens, vocabulary, how near the draft's distribution is to the target's
"""

import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _prompt(n, longest, heads, kv_heads, dim, dtype="bf16", ragged=True, causal=True, new=0, fused=False, pattern=0):
    return {"op": "prompt", "n": n, "longest": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "ragged": ragged, "causal": causal, "new": new, "fused": fused, "pattern": pattern}


def _cached(n, longest, heads, kv_heads, dim, dtype="bf16", page=16, tokens=1, prefix=0, members=1, ragged=True, pattern=0):
    return {"op": "cached", "n": n, "longest": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "page": page, "tokens": tokens, "prefix": prefix, "members": members, "ragged": ragged, "pattern": pattern}


def _pages(kind, n, longest, ways, pages, layers, kv_heads, dim, dtype="bf16", page=16, pattern=0):
    return {"op": "pages", "kind": kind, "n": n, "longest": longest, "ways": ways, "pages": pages, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "ragged": True, "pattern": pattern}


def _verify(n, drafts, vocab, dtype="fp32", close=0.5, ragged=False, pattern=0):
    return {"op": "verify", "n": n, "drafts": drafts, "vocab": vocab, "dtype": dtype, "close": close, "ragged": ragged,
            "pattern": pattern}


def listed():
    cases = [
        # one short question to a small decoder: launch and latency bound
        ("prompt 1x37 14/2x64", _prompt(1, 37, 14, 2, 64, ragged=False)),
        # requests that arrived together, of every length, some with nothing left to do; q, k, v from one product
        ("prompt 24 ragged 14/2x64", _prompt(24, 2048, 14, 2, 64, fused=True, pattern=1)),
        # the next 512 tokens of long prompts that are fed in pieces
        ("prompt 512 on 4608 32/8x128", _prompt(4, 4608, 32, 8, 128, "fp16", new=512, pattern=2)),
        # one long document
        ("prompt 1x16384 32/8x128", _prompt(1, 16384, 32, 8, 128, ragged=False)),
        # one user's chat, one token
        ("cached 1x200 14/2x64", _cached(1, 200, 14, 2, 64, ragged=False)),
        # a full batch of unrelated sequences, short and long, one token each
        ("cached 32x16384 32/8x128", _cached(32, 16384, 32, 8, 128, pattern=3)),
        # 64 requests on one long system prompt
        ("cached 64 on 8192 32/8x128", _cached(64, 8704, 32, 8, 128, prefix=8192, members=64, pattern=4)),
        # drafted tokens (and the one before them) of 16 sequences, 4 on each of 4 prompts
        ("cached 16x6 drafts 14/2x64", _cached(16, 2300, 14, 2, 64, "fp16", 64, tokens=6, prefix=1536, members=4, pattern=5)),
        # eight sampled answers to each of eight prompts: what each step of an answer's start does to the cache
        ("pages fork 8x8", _pages("fork", 8, 1500, 8, 2048, 24, 2, 64, pattern=6)),
        # a cache after many requests came and went
        ("pages compact 4096", _pages("compact", 40, 2000, 0, 4096, 24, 2, 64, pattern=7)),
        # one sequence, four drafts, a small vocabulary
        ("verify 1x4 v32000", _verify(1, 4, 32000)),
        # a batch, drafts of different lengths, a large odd vocabulary
        ("verify 64x7 v128003", _verify(64, 7, 128003, "bf16", 0.3, True, 8)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((14, 2), (32, 8), (16, 16), (8, 1), (28, 4), (12, 6))


def draw(rng):
    """One more case of the listed ranges: prompts of 1 to 16384 tokens, caches of 1 to 32768 tokens, batches of
    1 to 96, head sizes of 40 to 128, pages of 16 to 128 tokens, vocabularies of 500 to 160000."""
    pattern = rng.randrange(1 << 20)
    op = rng.choice(["prompt", "prompt", "cached", "cached", "cached", "pages", "verify"])
    heads, kv = rng.choice(HEADS)
    dim = rng.choice([64, 64, 128, 128, 80, 40, 112])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    limit = max(work(c)["flops"] for c in listed())
    if op == "prompt":
        while True:
            n, longest = _log(rng, 1, 48), _log(rng, 1, 16384)
            new = rng.choice([0, 0, 0, min(longest, _log(rng, 1, 1024))])
            c = _prompt(n, longest, heads, kv, dim, dtype, rng.random() < 0.7, rng.random() < 0.75, new,
                        new == 0 and rng.random() < 0.5, pattern)
            if work(c)["flops"] <= 0.5 * limit and n * longest <= 1 << 17:
                return c
    if op == "cached":
        while True:
            n, longest = _log(rng, 1, 96), _log(rng, 1, 32768)
            members, prefix = 1, 0
            if rng.random() < 0.5 and longest > 64:
                members, prefix = rng.randint(1, n), rng.randint(1, longest - 20)
            c = _cached(n, longest, heads, kv, dim, dtype, rng.choice([16, 16, 32, 64, 128]),
                        rng.choice([1, 1, 1, 2, 4, 5, 8, 16]), prefix, members, rng.random() < 0.8, pattern)
            if n * longest <= 1 << 19:
                return c
    if op == "pages":
        kind, page = rng.choice(["fork", "compact"]), rng.choice([16, 16, 32, 64])
        while True:
            layers, n, ways = rng.choice([1, 4, 12, 24]), _log(rng, 1, 32), rng.randint(1, 8)
            longest, kv, dim = _log(rng, 1, 2500), rng.choice([1, 2, 4]), rng.choice([64, 128])
            pages = n * (longest // page + 2) + n * ways * 2 + _log(rng, 1, 2048)
            if pages * page * layers * 4 * kv * dim <= 1 << 30:
                return _pages(kind, n, longest, ways, pages, layers, kv, dim, dtype, page, pattern)
    return _verify(_log(rng, 1, 64), rng.randint(1, 8), _log(rng, 500, 160000), rng.choice(["fp32", "bf16", "fp16"]),
                   rng.uniform(0.05, 1.0), rng.random() < 0.5, pattern)


# ---- what belongs to a case ----
def _lengths(case, least=0):
    """Tokens (keys) per sequence: the first has `longest`, the others fewer, over their logarithm, if ragged."""
    rng, n, top = random.Random(case["pattern"]), case["n"], case["longest"]
    if not case["ragged"]:
        return [top] * n
    low = max(1, least)
    lens = [top] + [_log(rng, low, max(low, top)) for _ in range(n - 1)]
    if least == 0 and n > 4:
        lens[n // 2] = 0
    return lens


def _prompt_lens(case):
    """(queries, keys) per sequence."""
    keys = _lengths(case)
    return [min(case["new"], m) if case["new"] else m for m in keys], keys


def _cached_lens(case):
    """(tokens held, valid queries) per sequence; every sequence holds its group's prefix."""
    least = case["prefix"] + 1 if case["members"] > 1 else 0
    lens = _lengths(case, least)
    rng = random.Random(case["pattern"] + 1)
    T = case["tokens"]
    return lens, [min(m, T if i % 3 else rng.randint(1, T)) for i, m in enumerate(lens)]


def _drafted(case):
    rng = random.Random(case["pattern"] + 2)
    return [rng.randint(0, case["drafts"]) if case["ragged"] and i else case["drafts"] for i in range(case["n"])]


def _pairs(n, m, causal):
    """Visible (query, key) pairs of n queries at the end of m keys."""
    if not causal:
        return n * m
    return sum(max(0, m - n + t + 1) for t in range(n))


def _page_lens(case):
    """Tokens of the live sequences of a page case."""
    return [max(1, m) for m in _lengths(case, 1)]


def _held_pages(case):
    """Pages of each live sequence, as ids in a pool where others came and went."""
    need = [-(-m // case["page"]) for m in _page_lens(case)]
    ids = random.Random(case["pattern"] + 3).sample(range(case["pages"]), sum(need))
    out, at = [], 0
    for c in need:
        out.append(ids[at:at + c])
        at += c
    return out


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "prompt":
        qs, ks = _prompt_lens(case)
        D, H, KV = case["dim"], case["heads"], case["kv_heads"]
        pairs = sum(_pairs(n, m, case["causal"]) for n, m in zip(qs, ks))
        return {"bytes": e * D * (2 * H * sum(qs) + 2 * KV * sum(ks)), "flops": 4 * D * H * pairs}
    if case["op"] == "cached":
        lens, valid = _cached_lens(case)
        D, H, KV, P, g = case["dim"], case["heads"], case["kv_heads"], case["prefix"], case["members"]
        shared = P // case["page"] * case["page"] if g > 1 else 0
        tokens = sum(m - shared for m in lens) + shared * -(-case["n"] // g)
        pairs = sum(_pairs(t, m, True) for t, m in zip(valid, lens))
        return {"bytes": e * D * (2 * KV * tokens + 2 * H * case["n"] * case["tokens"]), "flops": 4 * D * H * pairs}
    if case["op"] == "pages":
        page = case["layers"] * 2 * case["kv_heads"] * case["page"] * case["dim"] * e
        if case["kind"] == "compact":
            ids = [p for s in _held_pages(case) for p in s]
            moved = sum(p >= len(ids) for p in ids)
            return {"bytes": 2 * moved * page + 8 * len(ids) + 4 * case["pages"], "flops": moved}
        token = 2 * case["kv_heads"] * case["dim"] * e
        copies = sum(m % case["page"] > 0 for m in _page_lens(case)) * case["ways"]
        table = 4 * case["ways"] * sum(len(s) for s in _held_pages(case))
        return {"bytes": 2 * copies * page + 2 * case["n"] * case["ways"] * token + 2 * table, "flops": copies}
    # one row of p and of the noise per sequence, one of the draft's where something was rejected
    rows = sum(1 - (1 - 0.35 * case["close"]) ** k for k in _drafted(case))
    V = case["vocab"]
    return {"bytes": case["n"] * V * (e + 4) + rows * V * e, "flops": 2 * case["n"] * V}


# ---- inputs ----
def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 13)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=g.device) * scale).to(dtype)


def _offsets(lens, dev):
    return torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)


def _prepare_prompt(case, g, dev):
    qs, ks = _prompt_lens(case)
    H, KV, D, dt = case["heads"], case["kv_heads"], case["dim"], _DT[case["dtype"]]
    if case["fused"]:
        x = _normal(g, (sum(qs), (H + 2 * KV) * D), dt)
        x[:, :H * D] *= 2.0
        q, k, v = (t.unflatten(1, (-1, D)) for t in x.split([H * D, KV * D, KV * D], dim=1))
    else:
        q = _normal(g, (sum(qs), H, D), dt, 2.0)
        k, v = _normal(g, (sum(ks), KV, D), dt), _normal(g, (sum(ks), KV, D), dt)
    return {"q": q, "k": k, "v": v, "cu_q": _offsets(qs, dev), "cu_k": _offsets(ks, dev), "lens": (qs, ks)}


def _prepare_cached(case, g, dev):
    lens, valid = _cached_lens(case)
    page, P, m = case["page"], case["prefix"], case["members"]
    KV, D, dt = case["kv_heads"], case["dim"], _DT[case["dtype"]]
    rng = random.Random(case["pattern"] + 3)
    shared = P // page if m > 1 else 0                      # whole pages that a group's members have in common
    need = [-(-x // page) for x in lens]
    total = sum(need)                                       # an upper bound: members share pages
    ids = list(range(total + 7))
    rng.shuffle(ids)
    table = torch.full((case["n"], max(1, max(need))), -1, dtype=torch.int32)
    for i, c in enumerate(need):
        own_pages = [ids.pop() for _ in range(c)] if i % m == 0 else None
        if own_pages is None:
            first = table[i - i % m, :shared].tolist()
            own_pages = first + [ids.pop() for _ in range(c - shared)]
        table[i, :c] = torch.tensor(own_pages, dtype=torch.int32)
    pool = _normal(g, (total + 7, 1, 2, KV, page, D), dt)
    q = _normal(g, (case["n"], case["tokens"], case["heads"], D), dt, 2.0)
    groups = list(range(0, case["n"], m)) + [case["n"]]
    refs = torch.bincount(table[table >= 0].long(), minlength=total + 7).int()
    st = {"q": q, "pool": pool, "table": table.to(dev), "lens": torch.tensor(lens, dtype=torch.int32).to(dev),
          "refs": refs.to(dev), "seqs": torch.arange(case["n"], dtype=torch.int32).to(dev),
          "q_lens": torch.tensor(valid, dtype=torch.int32).to(dev),
          "groups": torch.tensor(groups, dtype=torch.int32).to(dev) if shared else None,
          "prefix_lens": torch.full((len(groups) - 1,), shared * page, dtype=torch.int32).to(dev) if shared else None,
          "host": (lens, valid)}
    if own:
        from tensorpack_amd.cache import PagedCache
        st["cache"] = PagedCache.from_buffers(pool, st["table"], st["lens"], st["refs"])
    return st


def _prepare_pages(case, g, dev):
    lens, held = _page_lens(case), _held_pages(case)
    page, n, ways = case["page"], case["n"], case["ways"] if case["kind"] == "fork" else 0
    width = max(len(s) for s in held) + 2
    table = torch.full((n * (1 + ways), width), -1, dtype=torch.int32)
    for i, s in enumerate(held):
        table[i, :len(s)] = torch.tensor(s, dtype=torch.int32)
    refs = torch.zeros(case["pages"], dtype=torch.int32)
    refs[torch.tensor([p for s in held for p in s])] = 1
    all_lens = torch.tensor(lens + [0] * (n * ways), dtype=torch.int32)
    dt, KV, D = _DT[case["dtype"]], case["kv_heads"], case["dim"]
    pool = _normal(g, (case["pages"], case["layers"], 2, KV, page, D), dt)
    st = {"pool": pool, "book": tuple(t.to(dev) for t in (table, all_lens, refs))}
    st["table"], st["lens"], st["refs"] = (t.clone() for t in st["book"])
    if ways:
        st["src"] = torch.arange(n, dtype=torch.int32).repeat_interleave(ways).to(dev)
        st["dst"] = torch.arange(n, n + n * ways, dtype=torch.int32).to(dev)
        st["counts"] = torch.ones(n * ways, dtype=torch.int32, device=dev)
        st["cu"] = torch.arange(n * ways + 1, dtype=torch.int32, device=dev)
        st["k"], st["v"] = _normal(g, (n * ways, KV, D), dt), _normal(g, (n * ways, KV, D), dt)
    if own:
        from tensorpack_amd.cache import PagedCache
        st["cache"] = PagedCache.from_buffers(pool, table.to(dev), all_lens.to(dev), refs.to(dev))
        st["snapshot"] = st["cache"].snapshot()
    return st


def _prepare_verify(case, g, dev):
    n, K, V, dt = case["n"], case["drafts"], case["vocab"], _DT[case["dtype"]]
    logits = torch.randn((n, K + 1, V), generator=g, device=dev) * 2.5
    p = torch.softmax(logits, -1).to(dt)
    logits[:, :K] += case["close"] * torch.randn((n, K, V), generator=g, device=dev)
    qf = torch.softmax(logits[:, :K], -1)
    race = 1.0 / torch.empty((n, K, V), device=dev).exponential_(generator=g).clamp_min(1e-20)
    drafts = (qf * race).argmax(-1).int()
    del race, logits
    noise = 1.0 / torch.empty((n, V), device=dev).exponential_(generator=g).clamp_min(1e-20)
    return {"p": p, "q": qf.to(dt), "drafts": drafts, "u": torch.rand((n, K), generator=g, device=dev), "noise": noise,
            "n_drafts": torch.tensor(_drafted(case), dtype=torch.int32).to(dev)}


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    make = {"prompt": _prepare_prompt, "cached": _prepare_cached, "pages": _prepare_pages, "verify": _prepare_verify}
    return dict(make[case["op"]](case, _gen(dev, seed), dev), case=case)


# ---- plain forms ----
def _softmax_rows(s):
    """exp(s - max) / sum over the last axis; rows of -inf alone give zeros."""
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _plain_attention(q, k, v, first, scale):
    """q (n, H, D), k and v (m, KV, D) in 32 bits; query t sees the first `first + t` keys (None: all)."""
    n, H, D = q.shape
    m, KV = k.shape[0], k.shape[1]
    out = torch.zeros_like(q)
    if m == 0 or n == 0:
        return out
    kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    step = max(1, (1 << 28) // (H * m))
    for a in range(0, n, step):
        b = min(n, a + step)
        rows = q[a:b].reshape(b - a, KV, H // KV, D).permute(1, 2, 0, 3).reshape(KV, -1, D)
        s = torch.matmul(rows, kt).view(KV, H // KV, b - a, m) * scale
        if first is not None:
            seen = torch.arange(m, device=q.device) < (torch.arange(a, b, device=q.device) + first)[:, None]
            s = torch.where(seen, s, -math.inf)
        o = torch.matmul(_softmax_rows(s).view(KV, -1, m), vt)
        out[a:b] = o.view(KV, H // KV, b - a, D).permute(2, 0, 1, 3).reshape(b - a, H, D)
    return out


def _plain_prompt(st):
    case, (qs, ks) = st["case"], st["lens"]
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    out, a, c = torch.empty_like(q), 0, 0
    for n, m in zip(qs, ks):
        out[a:a + n] = _plain_attention(q[a:a + n], k[c:c + m], v[c:c + m], m - n + 1 if case["causal"] else None,
                                        case["dim"] ** -0.5)
        a, c = a + n, c + m
    return out.to(st["q"].dtype)


def _plain_cached(st):
    case, (lens, valid) = st["case"], st["host"]
    out = torch.zeros(st["q"].shape, dtype=torch.float32, device=st["q"].device)
    for i, (m, t) in enumerate(zip(lens, valid)):
        if m == 0 or t == 0:
            continue
        pages = st["pool"][st["table"][i, :-(-m // case["page"])].long(), 0]         # (pages, 2, KV, page, D)
        kv = pages.permute(1, 0, 3, 2, 4).flatten(1, 2)[:, :m].float()
        out[i, :t] = _plain_attention(st["q"][i, :t].float(), kv[0], kv[1], m - t + 1, case["dim"] ** -0.5)
    return out.to(st["q"].dtype)


def _plain_free(st, seqs):
    rows = st["table"][seqs.long()]
    st["refs"].scatter_add_(0, rows.clamp(min=0).flatten().long(), -(rows >= 0).flatten().int())
    st["table"][seqs.long()] = -1
    st["lens"][seqs.long()] = 0


def _plain_fork(st, src, dst):
    rows = st["table"][src.long()]
    st["table"][dst.long()] = rows
    st["lens"][dst.long()] = st["lens"][src.long()]
    st["refs"].scatter_add_(0, rows.clamp(min=0).flatten().long(), (rows >= 0).flatten().int())


def _plain_extend(st, seqs, counts, page):
    """Pages for `counts` more tokens per sequence: the lowest free ids, in the sequences' order; a shared page
    that is partly filled is copied first."""
    s, table, refs, lens = seqs.long(), st["table"], st["refs"], st["lens"]
    have, more = lens[s].long(), counts.long()
    last = (have - 1).clamp(min=0) // page
    old = table[s, last].long()
    copy = (have % page > 0) & (more > 0) & (refs[old.clamp(min=0)] > 1)
    new = (have + more + page - 1) // page - (have + page - 1) // page
    need = new + copy
    start = need.cumsum(0) - need
    ids = torch.nonzero(refs == 0).flatten()[:int(need.sum())]
    row = torch.repeat_interleave(torch.arange(s.numel(), device=s.device), need)
    nth = torch.arange(row.numel(), device=s.device) - start[row]
    place = torch.where(copy[row] & (nth == 0), last[row], (have[row] + page - 1) // page + nth - copy[row].long())
    st["pool"][ids[start[copy]]] = st["pool"][old[copy]]
    refs.scatter_add_(0, old[copy], torch.full_like(old[copy], -1, dtype=torch.int32))
    refs[ids] = 1
    table[s[row], place] = ids.int()
    lens[s] += counts


def _plain_append(st, layer, k, v, seqs, cu, page):
    n = (cu[1:] - cu[:-1]).long()
    row = torch.repeat_interleave(seqs.long(), n)
    at = torch.arange(row.numel(), device=row.device) - torch.repeat_interleave(cu[1:].long(), n) + st["lens"][row].long()
    pages = st["table"][row, at // page].long()
    st["pool"][pages, layer, 0, :, at % page] = k.to(st["pool"].dtype)
    st["pool"][pages, layer, 1, :, at % page] = v.to(st["pool"].dtype)


def _plain_compact(st):
    """Pages in use take the lowest ids: those beyond move, in order, into the holes, in order."""
    refs, table = st["refs"], st["table"]
    used = refs > 0
    total = used.sum()
    ids = torch.arange(refs.numel(), device=refs.device)
    src, dst = torch.nonzero(used & (ids >= total)).flatten(), torch.nonzero(~used & (ids < total)).flatten()
    st["pool"][dst] = st["pool"][src]
    new = ids.clone()
    new[src] = dst
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()].int(), table))


def _plain_pages(st):
    case = st["case"]
    if case["kind"] == "compact":
        for t, s in zip((st["table"], st["lens"], st["refs"]), st["book"]):
            t.copy_(s)
        _plain_compact(st)
    else:
        _plain_free(st, st["dst"])
        _plain_fork(st, st["src"], st["dst"])
        _plain_extend(st, st["dst"], st["counts"], case["page"])
        _plain_append(st, 0, st["k"], st["v"], st["dst"], st["cu"], case["page"])
    return st["table"], st["lens"], st["refs"], st["pool"]


def _plain_verify(st):
    p, q, x, u = st["p"], st["q"], st["drafts"].long(), st["u"]
    n, K = x.shape
    px = p[:, :K].gather(2, x[:, :, None])[:, :, 0].float()
    qx = q.gather(2, x[:, :, None])[:, :, 0].float()
    j = torch.arange(K, device=x.device)
    good = (u * qx < px) & (j < st["n_drafts"][:, None])
    count = good.int().cumprod(1).sum(1)
    rows = torch.arange(n, device=x.device)
    w = p[rows, count].float()
    rest = torch.where((count < st["n_drafts"])[:, None], w - q[rows, count.clamp(max=K - 1)].float(), w).clamp(min=0)
    rest = torch.where((rest > 0).any(1, keepdim=True), rest, w)
    score = torch.where(rest > 0, rest * st["noise"], -1.0)
    best = score.amax(1, keepdim=True)
    first = torch.where(score == best, torch.arange(w.shape[1], device=x.device), w.shape[1]).amin(1)
    first = torch.where(best[:, 0] >= 0, first, -1)
    tokens = torch.full((n, K + 1), -1, dtype=st["drafts"].dtype, device=x.device)
    tokens[:, :K] = torch.where(j < count[:, None], st["drafts"], -1)
    tokens[rows, count] = first.to(tokens.dtype)
    return tokens, count.int()


# ---- the calls of a program ----
def _own_prompt(st):
    from tensorpack_amd.attention import prompt_attention
    return prompt_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], causal=st["case"]["causal"])


def _own_cached(st):
    from tensorpack_amd.attention import cached_attention
    return cached_attention(st["q"], st["cache"], 0, st["seqs"], q_lens=st["q_lens"], groups=st["groups"],
                            prefix_lens=st["prefix_lens"])


def _own_pages(st):
    cache = st["cache"]
    if st["case"]["kind"] == "compact":
        cache.restore(st["snapshot"])
        cache.compact()
    else:
        cache.free(st["dst"])
        cache.fork(st["src"], st["dst"])
        cache.extend(st["dst"], st["counts"])
        cache.append(0, st["k"], st["v"], st["dst"], st["cu"])
    return cache.table, cache.lens, cache.refs, cache.pool


def _own_verify(st):
    from tensorpack_amd.sampling import verify_drafts
    return verify_drafts(st["drafts"], st["p"], st["q"], st["u"], st["noise"], n_drafts=st["n_drafts"])


def run(state):
    plain = {"prompt": _plain_prompt, "cached": _plain_cached, "pages": _plain_pages, "verify": _plain_verify}
    calls = {"prompt": _own_prompt, "cached": _own_cached, "pages": _own_pages, "verify": _own_verify}
    return (calls if own else plain)[state["case"]["op"]](state)


# ---- 64 bits, from the definitions ----
def _exact_rows(q, k, v, visible, scale):
    """One head: q (n, D), k and v (m, D) double; row t sees the first visible[t] keys."""
    out = torch.zeros_like(q)
    m = k.shape[0]
    if m == 0:
        return out
    col = torch.arange(m, device=q.device)
    for a in range(0, q.shape[0], 2048):
        s = torch.mm(q[a:a + 2048], k.t().contiguous()).mul_(scale)
        s.masked_fill_(col[None, :] >= visible[a:a + 2048, None], -math.inf)
        w = torch.exp(s - s.amax(1, keepdim=True).clamp(min=-1e300))
        out[a:a + 2048] = torch.mm(w, v) / w.sum(1, keepdim=True).clamp(min=1e-300)
    return out


def _exact_prompt(case, st):
    qs, ks = _prompt_lens(case)
    G, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    a = c = 0
    for n, m in zip(qs, ks):
        t = torch.arange(n, device=out.device)
        visible = (t + 1 + m - n).clamp(min=0) if case["causal"] else torch.full_like(t, m)
        for h in range(case["heads"]):
            out[a:a + n, h] = _exact_rows(st["q"][a:a + n, h].double(), st["k"][c:c + m, h // G].double(),
                                          st["v"][c:c + m, h // G].double(), visible, scale)
        a, c = a + n, c + m
    return out


def _exact_cached(case, st):
    lens, valid = _cached_lens(case)
    page, G, T, D = case["page"], case["heads"] // case["kv_heads"], case["tokens"], case["dim"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    for i, m in enumerate(lens):
        t = valid[i]
        if m == 0 or t == 0:
            continue
        at = torch.arange(m, device=out.device)
        ids = st["table"][i].long()[at // page]
        visible = (torch.arange(t, device=out.device) + 1 + m - t).repeat_interleave(G)
        for g in range(case["kv_heads"]):
            k, v = (st["pool"][ids, 0, j, g, at % page].double() for j in (0, 1))
            rows = st["q"][i, :t, g * G:(g + 1) * G].double().reshape(t * G, D)
            out[i, :t, g * G:(g + 1) * G] = _exact_rows(rows, k, v, visible, D ** -0.5).view(t, G, D)
    return out


def _exact_pages(case, st):
    table, lens, refs = (t.tolist() for t in st["book"])
    pool, page = st["pool"].clone(), case["page"]
    if case["kind"] == "compact":
        live = [p for p, r in enumerate(refs) if r]
        holes = [p for p in range(len(live)) if not refs[p]]
        move = dict(zip([p for p in live if p >= len(live)], holes))
        for a, b in move.items():
            refs[b], refs[a] = refs[a], 0
            pool[b] = st["pool"][a]
        table = [[move.get(p, p) for p in row] for row in table]
    else:
        src, dst, kv = st["src"].tolist(), st["dst"].tolist(), (st["k"], st["v"])
        for a, b in zip(src, dst):
            table[b], lens[b] = list(table[a]), lens[a]
            for p in table[a]:
                if p >= 0:
                    refs[p] += 1
        free = iter([p for p, r in enumerate(refs) if r == 0])
        shared = [r > 1 for r in refs]
        for i, b in enumerate(dst):
            slot, off = lens[b] // page, lens[b] % page
            if off == 0:
                table[b][slot] = next(free)
                refs[table[b][slot]] = 1
            elif shared[table[b][slot]]:
                old, p = table[b][slot], next(free)
                pool[p] = st["pool"][old]
                refs[old], refs[p], table[b][slot] = refs[old] - 1, 1, p
            for j in (0, 1):
                pool[table[b][slot], 0, j, :, off] = kv[j][i]
            lens[b] += 1
    dev = pool.device
    return tuple(torch.tensor(t, dtype=torch.int32).to(dev) for t in (table, lens, refs)) + (pool,)


def _exact_verify(case, st):
    drafts, given = st["drafts"].tolist(), _drafted(case)
    n, K = case["n"], case["drafts"]
    tokens, counts = [[-1] * (K + 1) for _ in range(n)], []
    for i in range(n):
        took = 0
        while took < given[i]:
            x = drafts[i][took]
            if not float(st["u"][i, took]) * float(st["q"][i, took, x]) < float(st["p"][i, took, x]):
                break
            tokens[i][took] = x
            took += 1
        w = st["p"][i, took].double()
        if took < given[i]:
            d = (w - st["q"][i, took].double()).clamp(min=0)
            w = d if bool((d > 0).any()) else w
        s = (w * st["noise"][i].double()).cpu().numpy()
        tokens[i][took] = int(s.argmax()) if s.max() > 0 else -1
        counts.append(took)
    dev = st["p"].device
    return torch.tensor(tokens, dtype=torch.int32).to(dev), torch.tensor(counts, dtype=torch.int32).to(dev)


def exact(case, seed):
    if case["op"] in ("prompt", "cached") and work(case)["flops"] > 6e12:
        return None
    st = prepare(case, seed)
    f = {"prompt": _exact_prompt, "cached": _exact_cached, "pages": _exact_pages, "verify": _exact_verify}
    return f[case["op"]](case, st)
