"""Workloads of a decoder step's operators beside the 16-bit attention and cache, for timing and for comparing results.

  rotary  apply_rotary: positions into q and k
  store   QuantizedCache: new tokens quantised into the cache as they are written (append), then the newest tokens, or whole
          sequences, read back (read)
  attend  cached_attention over a QuantizedCache
  beam    beam_select over beams and vocabulary, and the cache's sequences reordered (PagedCache.reorder)

With `own` false, `run` computes them in plain torch operations (32 bits; 64 for angles and for scores next to each other),
rounded once at the end; with `own` true it makes the calls a program makes. Both get the same tensors from `prepare`.

Case fields
  op        rotary | store | attend | beam
  dtype     bf16 | fp16 | fp32: type of q, k, v or the logits
  heads, kv_heads, dim, page     shapes of attention and cache
  n         sequences (beam: prompts); longest: tokens of the longest; ragged: the others are shorter
  pattern   seed of what belongs to the case, not to the inputs: lengths, places of pages
  rows, rotated, interleaved, factor, original, far   (rotary) tokens, dims that turn, pairs side by side, stretch of the context,
            its first length (0: all frequencies are stretched alike), largest position
  layers, layer, new, window   (store) layers and the one written, new tokens per sequence, newest tokens read back (0: all)
  tokens, prefix, members      (attend) queries per sequence, tokens of a shared prefix, sequences per group
  ways, vocab, finished        (beam) beams per prompt, vocabulary, whether some beams have ended

The 8-bit pool: a page is [layers][K, V][kv_heads][page][dim up to a multiple of 16] codes of 8 bits, then
[layers][K, V][kv_heads][page / 16] scales in bf16, up to a multiple of 16 bytes; values are code * scale, scales powers of two.
"""

import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_RANGE = {"bf16": (-100, 100), "fp16": (-24, 9)}        # exponents of scales: code * 2**e is a number of the type
_BLOCK = 16


def _rotary(rows, heads, kv_heads, dim, rotated, dtype="bf16", interleaved=False, factor=1.0, original=0, far=4096, pattern=0):
    return {"op": "rotary", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotated": rotated, "dtype": dtype,
            "interleaved": interleaved, "factor": factor, "original": original, "far": far, "pattern": pattern}


def _store(n, longest, new, kv_heads, dim, dtype="bf16", page=16, layers=2, window=0, ragged=False, pattern=0):
    return {"op": "store", "n": n, "longest": longest, "new": new, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page,
            "layers": layers, "layer": layers - 1, "window": window, "ragged": ragged, "pattern": pattern}


def _attend(n, longest, heads, kv_heads, dim, dtype="bf16", page=16, tokens=1, prefix=0, members=1, ragged=True, pattern=0):
    return {"op": "attend", "n": n, "longest": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "page": page, "tokens": tokens, "prefix": prefix, "members": members, "ragged": ragged, "pattern": pattern}


def _beam(n, ways, vocab, longest, dtype="fp32", page=16, finished=False, pattern=0):
    return {"op": "beam", "n": n, "ways": ways, "vocab": vocab, "longest": longest, "dtype": dtype, "page": page,
            "finished": finished, "ragged": True, "pattern": pattern}


def listed():
    cases = [
        # one token of one sequence: launch and latency bound
        ("rotary 1 14/2x64", _rotary(1, 14, 2, 64, 64, far=1500)),
        # a prompt fed in one piece, far into a context stretched eightfold
        ("rotary 16384 32/8x128", _rotary(16384, 32, 8, 128, 128, factor=8.0, original=8192, far=65536, pattern=1)),
        # part of each head turned, pairs side by side, several requests' tokens
        ("rotary 2000 16/16x80 part", _rotary(2000, 16, 16, 80, 32, "fp16", True, far=4096, pattern=2)),
        # what each layer does to the cache for one token of a batch
        ("store 64 x 1 8x128", _store(64, 2000, 1, 8, 128, window=32, ragged=True, pattern=3)),
        # a long prompt into an empty cache
        ("store 1 x 16384 8x128", _store(1, 16384, 16384, 8, 128, page=64, window=0, pattern=4)),
        # the next piece of prompts that are fed in pieces: written, and all of them read for the attention of the piece
        ("store 4 x 512 on 4608 2x64", _store(4, 4608, 512, 2, 64, "fp16", ragged=True, pattern=5)),
        # one user's chat, one token
        ("attend 1x200 14/2x64", _attend(1, 200, 14, 2, 64, ragged=False)),
        # a full batch of unrelated sequences, short and long, one token each
        ("attend 32x16384 32/8x128", _attend(32, 16384, 32, 8, 128, pattern=6)),
        # 64 requests on one long system prompt
        ("attend 64 on 8192 32/8x128", _attend(64, 8704, 32, 8, 128, prefix=8192, members=64, pattern=7)),
        # drafted tokens (and the one before them) of 16 sequences, 4 on each of 4 prompts
        ("attend 16x6 drafts 14/2x64", _attend(16, 2300, 14, 2, 64, "fp16", 64, tokens=6, prefix=1536, members=4, pattern=8)),
        # one translation, four beams
        ("beam 1x4 v32000", _beam(1, 4, 32000, 120, pattern=9)),
        # a batch, a large odd vocabulary, some beams at their end
        ("beam 32x8 v128003", _beam(32, 8, 128003, 900, "bf16", finished=True, pattern=10)),
    ]
    return [dict(c, name=n) for n, c in cases]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((14, 2), (32, 8), (16, 16), (8, 1), (28, 4), (12, 6))


def draw(rng):
    """One more case of the listed ranges: 1 to 16384 rows turned or stored, caches of 1 to 32768 tokens, batches of 1 to 96,
    head sizes of 40 to 128, pages of 16 to 128 tokens, 1 to 16 beams over vocabularies of 500 to 160000."""
    pattern = rng.randrange(1 << 20)
    op = rng.choice(["rotary", "store", "store", "attend", "attend", "attend", "beam", "beam"])
    heads, kv = rng.choice(HEADS)
    dim = rng.choice([64, 64, 128, 128, 80, 40, 112])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rotary":
        while True:
            rows = _log(rng, 1, 16384)
            rotated = rng.choice([dim, dim, dim // 2, dim // 4])
            factor = rng.choice([1.0, 1.0, rng.uniform(1.5, 40.0)])
            c = _rotary(rows, heads, kv, dim, rotated, rng.choice([dtype, dtype, "fp32"]), rng.random() < 0.5, factor,
                        rng.choice([0, 2048, 8192]) if factor > 1 else 0, max(rows, _log(rng, 16, 1 << 20)), pattern)
            if work(c)["bytes"] <= 3.4e8:
                return c
    if op == "store":
        while True:
            n, longest = _log(rng, 1, 96), _log(rng, 1, 16384)
            new = rng.choice([1, 1, 2, 5, _log(rng, 1, longest), longest])
            c = _store(n, longest, min(new, longest), kv, dim, dtype, rng.choice([16, 16, 32, 64, 128]), rng.choice([1, 2, 4]),
                       rng.choice([0, new + _BLOCK]), rng.random() < 0.7, pattern)
            if n * longest * kv * dim <= 1 << 24:
                return c
    if op == "attend":
        while True:
            n, longest = _log(rng, 1, 96), _log(rng, 1, 32768)
            members, prefix = 1, 0
            if rng.random() < 0.5 and longest > 64:
                members, prefix = rng.randint(1, n), rng.randint(1, longest - 20)
            c = _attend(n, longest, heads, kv, dim, dtype, rng.choice([16, 16, 32, 64, 128]),
                        rng.choice([1, 1, 1, 2, 4, 5, 8, 16]), prefix, members, rng.random() < 0.8, pattern)
            if n * longest <= 1 << 19:
                return c
    while True:
        n, ways, vocab = _log(rng, 1, 64), rng.choice([1, 2, 3, 4, 4, 5, 8, 12, 16]), _log(rng, 500, 160000)
        if n * ways * vocab <= 32 * 8 * 128003:
            return _beam(n, ways, vocab, _log(rng, 1, 2000), rng.choice(["fp32", "bf16", "fp16"]), rng.choice([16, 32, 64]),
                         rng.random() < 0.5, pattern)


# ---- what belongs to a case ----
def _lengths(case, least=0):
    """Tokens per sequence: the first has `longest`, the others fewer, over their logarithm, if ragged."""
    rng, n, top = random.Random(case["pattern"]), case["n"], case["longest"]
    if not case["ragged"]:
        return [top] * n
    low = max(1, least)
    lens = [top] + [_log(rng, low, max(low, top)) for _ in range(n - 1)]
    if least == 0 and n > 4:
        lens[n // 2] = 0
    return lens


def _store_lens(case):
    """(tokens held in the end, new ones, tokens read back) per sequence."""
    lens = _lengths(case)
    new = [min(m, case["new"]) for m in lens]
    return lens, new, [min(m, case["window"] or m) for m in lens]


def _attend_lens(case):
    """(tokens held, valid queries) per sequence; every sequence holds its group's prefix."""
    least = case["prefix"] + 1 if case["members"] > 1 else 0
    lens = _lengths(case, least)
    rng = random.Random(case["pattern"] + 1)
    T = case["tokens"]
    return lens, [min(m, T if i % 3 else rng.randint(1, T)) for i, m in enumerate(lens)]


def _finished(case):
    rng = random.Random(case["pattern"] + 2)
    return [[case["finished"] and rng.random() < 0.2 for _ in range(case["ways"])] for _ in range(case["n"])]


def _tables(case, need, shared, members):
    """Page ids per sequence, in a pool where others came and went: need[i] pages, of which members of a group (`members`
    sequences in a row) have their first `shared` in common. Also the pages of the pool."""
    rng = random.Random(case["pattern"] + 3)
    total = sum(need) + 7
    ids = list(range(total))
    rng.shuffle(ids)
    rows = []
    for i, c in enumerate(need):
        first = rows[i - i % members][:shared] if i % members else []
        rows.append(first + [ids.pop() for _ in range(c - len(first))])
    width = max(1, max(need))
    return torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32), total


def _beam_rows(case):
    """Tokens of each beam's sequence; the beams of a prompt are of one length."""
    return [m for m in _lengths(case, 1) for _ in range(case["ways"])]


def _pairs(n, m):
    """Visible (query, key) pairs of n queries at the end of m keys."""
    return sum(max(0, m - n + t + 1) for t in range(n))


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "rotary":
        heads = case["heads"] + case["kv_heads"]
        return {"bytes": case["rows"] * (2 * heads * case["dim"] * e + 4), "flops": 3 * case["rows"] * heads * case["rotated"]}
    if case["op"] == "store":
        lens, new, back = _store_lens(case)
        per, D = 2 * case["kv_heads"], case["dim"]
        # rows in and codes out, then codes in and rows out; a scale per 16 tokens both times
        b = per * D * (e + 1) * (sum(new) + sum(back)) + per * 2 * (sum(new) + sum(back)) // _BLOCK
        return {"bytes": b, "flops": 2 * per * D * (sum(new) + sum(back))}
    if case["op"] == "attend":
        lens, valid = _attend_lens(case)
        D, H, KV, P, g = case["dim"], case["heads"], case["kv_heads"], case["prefix"], case["members"]
        shared = P // case["page"] * case["page"] if g > 1 else 0
        tokens = sum(m - shared for m in lens) + shared * -(-case["n"] // g)
        pairs = sum(_pairs(t, m) for t, m in zip(valid, lens))
        return {"bytes": 2 * KV * tokens * D + 4 * KV * tokens // _BLOCK + e * D * 2 * H * case["n"] * case["tokens"],
                "flops": 4 * D * H * pairs}
    live = sum(not f for row in _finished(case) for f in row)
    pages = sum(-(-m // case["page"]) for m in _beam_rows(case))
    return {"bytes": live * case["vocab"] * e + 16 * case["n"] * case["ways"] + 8 * pages, "flops": 4 * live * case["vocab"]}


# ---- the 8-bit pool ----
def _page_bytes(layers, kv_heads, page, dim):
    b = layers * 2 * kv_heads * (page * (-(-dim // 16) * 16) + page // _BLOCK * 2)
    return -(-b // 16) * 16


def _views(pool, layers, kv_heads, page, dim):
    """(codes (pages, layers, 2, kv_heads, page, dim) int8, scales (pages, layers, 2, kv_heads, page / 16) bf16) of a pool."""
    n, room = pool.shape[0], -(-dim // 16) * 16
    codes = pool[:, :layers * 2 * kv_heads * page * room].view(n, layers, 2, kv_heads, page, room)[..., :dim]
    at = layers * 2 * kv_heads * page * room
    scales = pool[:, at:at + layers * 4 * kv_heads * (page // _BLOCK)].view(torch.bfloat16)
    return codes, scales.view(n, layers, 2, kv_heads, page // _BLOCK)


def _exponents(top, dtype):
    """The smallest e with top <= 127 * 2**e, within the type's range."""
    m, e = torch.frexp(top)
    e = torch.where(m <= 127 / 128, e - 7, e - 6)
    lo, hi = _RANGE[dtype]
    return torch.where(top > 0, e, lo).clamp(lo, hi)


def _power(e):
    """2**e in 32 bits, put together from its bits (a library's power may round)."""
    return ((e.int().clamp(-126, 127) + 127) << 23).view(torch.float32)


def _codes(x, e):
    return torch.round(x * _power(-e)).clamp(-127, 127)


def _quantize_pages(x, dtype):
    """Whole blocks: (codes, scales) of x (..., page, dim)."""
    blocks = x.float().unflatten(-2, (-1, _BLOCK))
    e = _exponents(blocks.abs().amax((-1, -2)), dtype)
    codes = _codes(blocks, e[..., None, None]).to(torch.int8).flatten(-3, -2)
    return codes, _power(e).bfloat16()


# ---- inputs ----
def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 13)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=g.device) * scale).to(dtype)


def _offsets(lens, dev):
    return torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)


def _frequencies(case):
    rd, f = case["rotated"], []
    for i in range(rd // 2):
        x = 10000.0 ** (-2 * i / rd)
        if case["factor"] > 1:
            keep = 0.0                                  # slow dims are stretched, those that turn often are not
            if case["original"]:
                keep = min(1.0, max(0.0, (case["original"] * x / (2 * math.pi) - 1.0) / 3.0))
            x *= keep + (1 - keep) / case["factor"]
        f.append(x)
    return f


def _prepare_rotary(case, g, dev):
    H, KV, D, rows = case["heads"], case["kv_heads"], case["dim"], case["rows"]
    x = _normal(g, (rows, (H + 2 * KV) * D), _DT[case["dtype"]])
    q, k, _ = (t.unflatten(1, (-1, D)) for t in x.split([H * D, KV * D, KV * D], dim=1))
    first = torch.randint(0, max(1, case["far"] - rows + 1), (1,), generator=g, device=dev, dtype=torch.int32)
    st = {"q": q, "k": k, "positions": first + torch.arange(rows, dtype=torch.int32, device=dev),
          "frequencies": torch.tensor(_frequencies(case), dtype=torch.float64).to(dev)}
    if own:
        from tensorpack_amd.rotary import Rotary
        st["rotary"] = Rotary(case["rotated"], interleaved=case["interleaved"], factor=case["factor"],
                              original=case["original"] or None, device=dev)
    return st


def _prepare_store(case, g, dev):
    lens, new, back = _store_lens(case)
    L, KV, D, page, dt = case["layers"], case["kv_heads"], case["dim"], case["page"], _DT[case["dtype"]]
    table, pages = _tables(case, [-(-m // page) for m in lens], 0, 1)
    pool = torch.zeros((pages, _page_bytes(L, KV, page, D)), dtype=torch.int8, device=dev)
    codes, scales = _views(pool, L, KV, page, D)
    # tokens differ in size, so that a block's scale can grow with a new one
    x = torch.randn((pages, 2, KV, page, D), generator=g, device=dev)
    x *= torch.exp(0.5 * torch.randn((pages, 2, 1, page, 1), generator=g, device=dev))
    c, s = _quantize_pages(x, case["dtype"])
    codes[:, case["layer"]], scales[:, case["layer"]] = c, s
    rows = sum(new)
    k, v = (_normal(g, (rows, KV, D), torch.float32) * torch.exp(0.5 * torch.randn((rows, 1, 1), generator=g, device=dev)) for _ in (0, 1))
    held = torch.tensor(lens, dtype=torch.int32).to(dev)
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).int().to(dev)
    st = {"pool": pool, "start": pool.clone(), "k": k.to(dt), "v": v.to(dt), "table": table.to(dev), "lens": held,
          "seqs": torch.arange(case["n"], dtype=torch.int32).to(dev), "cu": _offsets(new, dev), "cu_back": _offsets(back, dev),
          "rows_back": sum(back)}
    if own:
        from tensorpack_amd.cache import QuantizedCache
        st["cache"] = QuantizedCache.from_buffers(pool, st["table"], held, refs, n_layers=L, n_kv_heads=KV, head_dim=D,
                                                  page_size=page, dtype=dt)
    return st


def _prepare_attend(case, g, dev):
    lens, valid = _attend_lens(case)
    page, P, m = case["page"], case["prefix"], case["members"]
    KV, D, dt = case["kv_heads"], case["dim"], _DT[case["dtype"]]
    shared = P // page if m > 1 else 0                      # whole pages that a group's members have in common
    table, pages = _tables(case, [-(-x // page) for x in lens], shared, m)
    pool = torch.zeros((pages, _page_bytes(1, KV, page, D)), dtype=torch.int8, device=dev)
    codes, scales = _views(pool, 1, KV, page, D)
    for i in range(0, pages, 4096):
        c, s = _quantize_pages(torch.randn((min(pages - i, 4096), 1, 2, KV, page, D), generator=g, device=dev), case["dtype"])
        codes[i:i + 4096], scales[i:i + 4096] = c, s
    q = _normal(g, (case["n"], case["tokens"], case["heads"], D), dt, 2.0)
    groups = list(range(0, case["n"], m)) + [case["n"]]
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).int().to(dev)
    st = {"q": q, "pool": pool, "table": table.to(dev), "lens": torch.tensor(lens, dtype=torch.int32).to(dev),
          "seqs": torch.arange(case["n"], dtype=torch.int32).to(dev), "q_lens": torch.tensor(valid, dtype=torch.int32).to(dev),
          "groups": torch.tensor(groups, dtype=torch.int32).to(dev) if shared else None,
          "prefix_lens": torch.full((len(groups) - 1,), shared * page, dtype=torch.int32).to(dev) if shared else None}
    if own:
        from tensorpack_amd.cache import QuantizedCache
        st["cache"] = QuantizedCache.from_buffers(pool, st["table"], st["lens"], refs, n_layers=1, n_kv_heads=KV, head_dim=D,
                                                  page_size=page, dtype=dt)
    return st


def _prepare_beam(case, g, dev):
    n, W, V, page = case["n"], case["ways"], case["vocab"], case["page"]
    logits = (torch.randn((n, W, V), generator=g, device=dev) * 2.5).to(_DT[case["dtype"]])
    scores = -40.0 * torch.rand((n, 1), generator=g, device=dev) - 3.0 * torch.rand((n, W), generator=g, device=dev)
    lens = _beam_rows(case)
    shared = min(lens) // page // 2
    table, pages = _tables(case, [-(-m // page) for m in lens], shared, W)
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).int()
    book = tuple(t.to(dev) for t in (table, torch.tensor(lens, dtype=torch.int32), refs))
    st = {"logits": logits, "scores": scores, "done": torch.tensor(_finished(case)).to(dev), "book": book,
          "seqs": torch.arange(n * W, dtype=torch.int32).to(dev)}
    st["table"], st["lens"], st["refs"] = (t.clone() for t in book)
    if own:
        from tensorpack_amd.cache import PagedCache
        pool = torch.zeros((pages, 1, 2, 1, page, 8), dtype=torch.bfloat16, device=dev)
        st["cache"] = PagedCache.from_buffers(pool, *book)
        st["snapshot"] = st["cache"].snapshot()
    return st


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    make = {"rotary": _prepare_rotary, "store": _prepare_store, "attend": _prepare_attend, "beam": _prepare_beam}
    return dict(make[case["op"]](case, _gen(dev, seed), dev), case=case)


# ---- plain forms ----
def _plain_turn(x, cos, sin, rd, interleaved):
    y = x.float()
    t = y[..., :rd]
    a, b = (t[..., 0::2], t[..., 1::2]) if interleaved else (t[..., :rd // 2], t[..., rd // 2:])
    both = (a * cos - b * sin, a * sin + b * cos)
    t = torch.stack(both, -1).flatten(-2) if interleaved else torch.cat(both, -1)
    return torch.cat((t, y[..., rd:]), -1).to(x.dtype)


def _plain_rotary(st):
    case = st["case"]
    turn = st["positions"].double()[:, None, None] * st["frequencies"]
    cos, sin = torch.cos(turn).float(), torch.sin(turn).float()
    return tuple(_plain_turn(st[x], cos, sin, case["rotated"], case["interleaved"]) for x in ("q", "k"))


def _plain_places(st, cu):
    """(sequence, place in it) of each row: rows cu[i]:cu[i + 1] are the last tokens of sequence i."""
    n = (cu[1:] - cu[:-1]).long()
    row = torch.repeat_interleave(st["seqs"].long(), n, output_size=st["rows"])
    end = torch.repeat_interleave(cu[1:].long(), n, output_size=st["rows"])
    return row, torch.arange(st["rows"], device=row.device) - end + st["lens"][row].long()


def _plain_append(st, codes, scales):
    """New tokens into the blocks that they fall into: a block's scale is the larger of its old tokens' and its new ones', and
    old codes are rounded to it."""
    case = st["case"]
    page, layer, lo = case["page"], case["layer"], _RANGE[case["dtype"]][0]
    st["rows"] = st["k"].shape[0]
    seq, at = _plain_places(st, st["cu"])
    x = torch.stack((st["k"], st["v"]), 1).float()                                   # (rows, 2, KV, D)
    per = page // _BLOCK
    number, of = torch.unique(st["table"][seq, at // page].long() * per + at % page // _BLOCK, return_inverse=True)
    ids, block = number // per, number % per                                         # the blocks that get tokens
    top = torch.zeros((number.numel(),) + tuple(x.shape[1:3]), device=x.device)
    top.scatter_reduce_(0, of[:, None, None].expand(x.shape[:3]), x.abs().amax(-1), "amax")
    first = torch.full((number.numel(),), _BLOCK, dtype=torch.long, device=x.device)
    first.scatter_reduce_(0, of, at % _BLOCK, "amin")
    old = torch.frexp(scales[ids, layer, :, :, block].float())[1] - 1
    e = torch.maximum(_exponents(top, case["dtype"]), torch.where((first > 0)[:, None, None], old, lo))
    places = block[:, None] * _BLOCK + torch.arange(_BLOCK, device=x.device)
    held = codes[ids[:, None], layer, :, :, places].float()                          # (blocks, 16, 2, KV, D)
    held = _codes(held, (e - old)[:, None, :, :, None])
    held[of, at % _BLOCK] = _codes(x, e[of][..., None])
    codes[ids[:, None], layer, :, :, places] = held.to(torch.int8)
    scales[ids, layer, :, :, block] = _power(e).bfloat16()


def _plain_read(st, codes, scales):
    case = st["case"]
    page, layer = case["page"], case["layer"]
    st["rows"] = st["rows_back"]
    seq, at = _plain_places(st, st["cu_back"])
    pages = st["table"][seq, at // page].long()
    x = codes[pages, layer, :, :, at % page].float() * scales[pages, layer, :, :, at % page // _BLOCK].float()[..., None]
    x = x.to(_DT[case["dtype"]])
    return x[:, 0].contiguous(), x[:, 1].contiguous()


def _plain_store(st):
    case = st["case"]
    codes, scales = _views(st["pool"], case["layers"], case["kv_heads"], case["page"], case["dim"])
    _plain_append(st, codes, scales)
    return _plain_read(st, codes, scales)


def _plain_attend(st):
    case = st["case"]
    n, T, H, D = st["q"].shape
    KV, page = case["kv_heads"], case["page"]
    codes, scales = _views(st["pool"], 1, KV, page, D)
    ids = st["table"].clamp(min=0).long()                                             # (n, pages)
    m = ids.shape[1] * page

    def values(i):                                                                    # (n, KV, m, D)
        x = codes[ids, 0, i].float().unflatten(3, (-1, _BLOCK)) * scales[ids, 0, i].float()[..., None, None]
        return x.flatten(3, 4).transpose(1, 2).reshape(n, KV, m, D)
    rows = st["q"].float().view(n, T, KV, H // KV, D).permute(0, 2, 1, 3, 4).reshape(n, KV, -1, D)
    s = torch.matmul(rows, values(0).transpose(2, 3).contiguous()).view(n, KV, T, H // KV, m) * D ** -0.5
    t = torch.arange(T, device=s.device)
    seen = torch.where(t < st["q_lens"][:, None], st["lens"][:, None] - st["q_lens"][:, None] + t + 1, 0)     # (n, T)
    s = torch.where(torch.arange(m, device=s.device) < seen[:, None, :, None, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, 1.0, total)
    o = torch.matmul(w.view(n, KV, -1, m), values(1)).view(n, KV, T, H // KV, D)
    return o.permute(0, 2, 1, 3, 4).reshape(n, T, H, D).to(st["q"].dtype)


def _plain_beam(st):
    n, W, V = st["logits"].shape
    x = st["logits"].double()
    top = x.amax(-1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    x = torch.where(st["done"][..., None], -math.inf, x)
    x[..., 0] = torch.where(st["done"], 0.0, x[..., 0])                               # an ended beam stands as it is, token 0
    x = (x + st["scores"].double()[..., None]).view(n, W * V)
    best, at = torch.sort(x, dim=1, descending=True, stable=True)
    best, at = best[:, :W], at[:, :W]
    parents = (at // V + W * torch.arange(n, device=at.device)[:, None]).int()
    for t, s in zip((st["table"], st["lens"], st["refs"]), st["book"]):
        t.copy_(s)
    seqs, src = st["seqs"].long(), st["seqs"].long()[parents.flatten().long()]
    before, rows = st["table"][seqs], st["table"][src]
    st["refs"].scatter_add_(0, rows.clamp(min=0).flatten().long(), (rows >= 0).flatten().int())
    st["refs"].scatter_add_(0, before.clamp(min=0).flatten().long(), -(before >= 0).flatten().int())
    st["lens"][seqs] = st["lens"][src]
    st["table"][seqs] = rows
    return best.float(), (at % V).int(), parents, st["table"], st["lens"], st["refs"]


# ---- the calls of a program ----
def _own_rotary(st):
    from tensorpack_amd.rotary import apply_rotary
    return apply_rotary(st["rotary"], st["q"], st["k"], st["positions"])


def _own_store(st):
    cache, layer = st["cache"], st["case"]["layer"]
    cache.append(layer, st["k"], st["v"], st["seqs"], st["cu"])
    return cache.read(layer, st["seqs"], st["cu_back"], st["rows_back"])


def _own_attend(st):
    from tensorpack_amd.attention import cached_attention
    return cached_attention(st["q"], st["cache"], 0, st["seqs"], q_lens=st["q_lens"], groups=st["groups"],
                            prefix_lens=st["prefix_lens"])


def _own_beam(st):
    from tensorpack_amd.sampling import beam_select
    cache = st["cache"]
    scores, tokens, parents = beam_select(st["logits"], st["scores"], done=st["done"])
    cache.restore(st["snapshot"])
    cache.reorder(st["seqs"], parents.view(-1))
    return scores, tokens, parents, cache.table, cache.lens, cache.refs


def run(state):
    plain = {"rotary": _plain_rotary, "store": _plain_store, "attend": _plain_attend, "beam": _plain_beam}
    calls = {"rotary": _own_rotary, "store": _own_store, "attend": _own_attend, "beam": _own_beam}
    return (calls if own else plain)[state["case"]["op"]](state)


# ---- 64 bits, from the definitions ----
def _exact_rotary(case, st):
    rd = case["rotated"]
    out = []
    for x in (st["q"].double(), st["k"].double()):
        y = x.clone()
        for i, f in enumerate(_frequencies(case)):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rd // 2)
            z = torch.polar(torch.ones_like(x[:, 0, 0]), st["positions"].double() * f)[:, None] * torch.complex(x[..., a], x[..., b])
            y[..., a], y[..., b] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_store(case, st):
    lens, new, back = _store_lens(case)
    page, D, layer = case["page"], case["dim"], case["layer"]
    lo, hi = _RANGE[case["dtype"]]
    codes, scales = _views(st["start"], case["layers"], case["kv_heads"], page, D)
    codes, scales = codes[:, layer].double(), scales[:, layer].double()
    out, row = ([], []), 0
    for i, m in enumerate(lens):
        blocks = -(-m // _BLOCK)
        if not blocks:
            continue
        at = torch.arange(blocks, device=codes.device) * _BLOCK
        ids, within = st["table"][i].long()[at // page], at % page // _BLOCK
        took = row + new[i]
        for j, x in enumerate((st["k"], st["v"])):
            # (blocks, heads, 16, D): what the blocks hold, then with the new tokens in their places
            old_scale = scales[ids, j, :, within]
            held = codes[ids, j].unflatten(2, (-1, _BLOCK))[torch.arange(blocks), :, within] * old_scale[..., None, None]
            fresh = torch.zeros((blocks * _BLOCK,) + tuple(x.shape[1:]), dtype=torch.float64, device=x.device)
            fresh[m - new[i]:m] = x[row:took].double()
            fresh = fresh.unflatten(0, (blocks, _BLOCK)).transpose(1, 2)
            place = at[:, None] + torch.arange(_BLOCK, device=at.device)
            is_new = (place >= m - new[i]) & (place < m)
            large = (fresh * is_new[:, None, :, None]).abs().amax((2, 3))
            e = torch.ceil(torch.log2(large / 127.0).nan_to_num(neginf=-500.0)).clamp(-500, 500)
            for step in (1, -1):                        # the logarithm may be off by its rounding
                moved = large > 127.0 * _exact_power(e) if step > 0 else large <= 127.0 * _exact_power(e - 1)
                e = torch.where(moved, e + step, e)
            e = e.clamp(lo, hi)
            before = torch.log2(old_scale).round()
            kept = (place[:, 0] < m - new[i])[:, None]
            e = torch.where(kept, torch.maximum(e, before), e)
            e = _exact_power(torch.where(is_new.any(1)[:, None], e, before))[..., None, None]
            y = torch.where(is_new[:, None, :, None], fresh, held)
            y = (y / e).round().clamp(-127, 127) * e
            out[j].append(y.transpose(1, 2).flatten(0, 1)[m - back[i]:m])
        row = took
    return tuple(torch.cat(x) if x else torch.zeros((0, case["kv_heads"], D), dtype=torch.float64, device=codes.device) for x in out)


def _exact_attend(case, st):
    lens, valid = _attend_lens(case)
    page, G, T, D = case["page"], case["heads"] // case["kv_heads"], case["tokens"], case["dim"]
    codes, scales = _views(st["pool"], 1, case["kv_heads"], page, D)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    for i, m in enumerate(lens):
        t = valid[i]
        if m == 0 or t == 0:
            continue
        at = torch.arange(m, device=out.device)
        ids = st["table"][i].long()[at // page]
        visible = (torch.arange(t, device=out.device) + 1 + m - t).repeat_interleave(G)
        for g in range(case["kv_heads"]):
            k, v = (codes[ids, 0, j, g, at % page].double() * scales[ids, 0, j, g, at % page // _BLOCK].double()[:, None] for j in (0, 1))
            rows = st["q"][i, :t, g * G:(g + 1) * G].double().reshape(t * G, D)
            s = torch.mm(rows, k.t().contiguous()) / math.sqrt(D)
            s.masked_fill_(at[None, :] >= visible[:, None], -math.inf)
            p = torch.exp(s - s.amax(1, keepdim=True))
            out[i, :t, g * G:(g + 1) * G] = (torch.mm(p, v) / p.sum(1, keepdim=True)).view(t, G, D)
    return out


def _exact_beam(case, st):
    n, W, V = st["logits"].shape
    done, start = _finished(case), st["scores"].tolist()
    scores, tokens, parents = [], [], []
    for b in range(n):
        rows = []
        for w in range(W):
            if done[b][w]:
                rows.append((torch.tensor([start[b][w]], dtype=torch.float64), torch.tensor([0]), w))
                continue
            x = st["logits"][b, w].double()
            x = x - torch.logsumexp(x, 0)
            # every value that could be among the W best, in index order
            keep = torch.nonzero(x >= torch.topk(x, min(W, V)).values[-1]).flatten()
            rows.append(((x[keep] + start[b][w]).cpu(), keep.cpu(), w))
        found = sorted(((-float(s), w, int(t)) for c, ts, w in rows for s, t in zip(c, ts)))[:W]
        scores.append([-s for s, _, _ in found])
        tokens.append([t for _, _, t in found])
        parents.append([b * W + w for _, w, _ in found])
    table, lens, refs = (t.tolist() for t in st["book"])
    flat = [p for row in parents for p in row]
    after = [list(table[p]) for p in flat]
    for old, fresh in zip(table, after):
        for p in fresh:
            refs[p] += p >= 0
        for p in old:
            refs[p] -= p >= 0
    dev = st["logits"].device
    whole = tuple(torch.tensor(t, dtype=torch.int32).to(dev) for t in (tokens, parents, after, [lens[p] for p in flat], refs))
    return (torch.tensor(scores, dtype=torch.float64).to(dev),) + whole


def exact(case, seed):
    st = prepare(case, seed)
    f = {"rotary": _exact_rotary, "store": _exact_store, "attend": _exact_attend, "beam": _exact_beam}
    return f[case["op"]](case, st)
