"""Attention where one key takes nearly all the weight and what is left matters, against 64 bits.

Bar, per element, with u the unit roundoff of the 16-bit type and A = sum_j w_j |v_j|: a weight and the result are each rounded
once (u A + u |o|), fp32 steps 2^-14 A, the type's smallest value. In f16 a weight also has the type's range: the kernels place the
row's largest between 2^7 and 2^15, so that each weight loses less than 2^-25 / 2^7 = 2^-32 of it besides: 2^-32 sum_j |v_j|."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
DIM = 64


def _ints(x, dev):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _case(keys, sink, gap, values):
    """k and v (keys, DIM): scores of 0 but for the sink's, `gap` above; v: `values` at each key, 0 at the sink."""
    k, v = np.zeros((keys, DIM), np.float32), np.zeros((keys, DIM), np.float32)
    k[sink, 0] = gap
    v[:] = np.resize(np.asarray(values, np.float32), keys)[:, None]
    v[sink] = 0
    return k, v


def _check(got, k, v, dtype):
    u, tiny, lost = (2.0 ** -8, 2.0 ** -133, 0.0) if dtype == "bf16" else (2.0 ** -11, 2.0 ** -24, 2.0 ** -32)
    s = k[:, 0].astype(np.float64)
    w = np.exp(s - s.max())
    w /= w.sum()
    o, A = w @ v.astype(np.float64), w @ np.abs(v.astype(np.float64))
    bar = u * (A + np.abs(o)) + 2.0 ** -14 * A + tiny + lost * np.abs(v.astype(np.float64)).sum(0)
    assert (np.abs(o) > 4 * bar).any()                           # an answer of 0 would not do
    err = np.abs(got.double().cpu().numpy().reshape(-1, DIM) - o)
    assert (err <= bar).all(), (err.max(), bar.min(), o.max())


CASES = {"one weak key": (18.0, [1000.0] + [0.0] * 10 ** 6), "many weaker keys": (14.0, [1.0]), "ten bits down": (7.0, [3.0, 1.0, 0.5])}


@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,keys,at_end", [(1, 100, 0), (40, 900, 0), (40, 900, 1), (3, 4000, 0), (3, 4000, 1), (400, 700, 1)])
def test_prompt(gpu, case, dtype, rows, keys, at_end):
    import torch
    from tensorpack_amd.attention import prompt_attention
    print(case, dtype, rows, keys, at_end, flush=True)
    dt = torch.float16 if dtype == "fp16" else torch.bfloat16
    k, v = _case(keys, keys - 1 if at_end else 5, *CASES[case])
    q = torch.zeros((rows, 2, DIM), dtype=dt, device=gpu)
    q[..., 0] = 8.0                                              # times 1/8: the scores are k[:, 0]
    up = lambda x: torch.from_numpy(x).to(gpu, dt)[:, None].contiguous()
    got = prompt_attention(q, up(k), up(v), _ints([0, rows], gpu), _ints([0, keys], gpu), causal=False)
    _check(got, k, v, dtype)


@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,prefix", [(2, 0), (20, 0), (40, 0), (2, 640), (40, 640)])
@pytest.mark.parametrize("at_end", [0, 1])
def test_cached(gpu, case, dtype, heads, prefix, at_end):
    import torch
    from tensorpack_amd.attention import cached_attention
    from tensorpack_amd.cache import PagedCache
    print(case, dtype, heads, prefix, at_end, flush=True)
    dt, keys = torch.float16 if dtype == "fp16" else torch.bfloat16, 1500
    k, v = _case(keys, keys - 1 if at_end else 5, *CASES[case])
    cache = PagedCache(200, 1, 1, DIM, max_seqs=2, max_pages=100, dtype=dt, device=gpu)
    cache.extend(_ints([0], gpu), _ints([keys], gpu))
    up = lambda x: torch.from_numpy(x).to(gpu, dt)[:, None].contiguous()
    cache.append(0, up(k), up(v), _ints([0], gpu), _ints([0, keys], gpu))
    cache.fork(_ints([0], gpu), _ints([1], gpu))
    q = torch.zeros((2, 1, heads, DIM), dtype=dt, device=gpu)
    q[..., 0] = 8.0
    kw = {"groups": _ints([0, 2], gpu), "prefix_lens": _ints([prefix], gpu)} if prefix else {}
    _check(cached_attention(q, cache, 0, _ints([0, 1], gpu), **kw), k, v, dtype)
    cache.check()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("heads", [1, 20, 40])                   # 16, 32 and more rows: each has a way of its own
@pytest.mark.parametrize("keys", [2, 40, 200])
def test_cached_weights_add_up(gpu, dtype, heads, keys):
    """A constant V comes out as it is: the weights that are summed are those that V is multiplied with, so their rounding drops
    out. All weights but one lie just below the middle of two values of the type (all round down, by nearly u of each), and
    V has the largest mantissa, whose half unit is u / 2 of it. With agreeing sums each weight times v and each sum is an fp32
    rounding (2^-24 for each of 200 keys: under 2^-16 of the result), far below that half unit."""
    import torch
    from tensorpack_amd.attention import cached_attention
    from tensorpack_amd.cache import PagedCache
    print(dtype, heads, keys, flush=True)
    dt, u = (torch.float16, 2.0 ** -11) if dtype == "fp16" else (torch.bfloat16, 2.0 ** -8)
    cache = PagedCache(30, 1, 1, DIM, max_seqs=1, max_pages=20, dtype=dt, device=gpu)
    cache.extend(_ints([0], gpu), _ints([keys], gpu))
    k = torch.zeros((keys, 1, DIM), dtype=dt, device=gpu)
    k[1:, 0, 0] = -1.0
    v = torch.full((keys, 1, DIM), 2.0 - 2.0 * u, dtype=dt, device=gpu)
    cache.append(0, k, v, _ints([0], gpu), _ints([0, keys], gpu))
    q = torch.zeros((1, 1, heads, DIM), dtype=dt, device=gpu)
    q[..., 0] = 1.0
    scale = float(np.log(2.0) - np.log1p(0.9 * u))               # weights 1 and 1/2 + 0.45 u
    got = cached_attention(q, cache, 0, _ints([0], gpu), scale=scale)
    assert torch.equal(got, v[:1].expand(1, 1, heads, DIM))
