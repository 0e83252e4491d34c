"""Attention between the q/k/v and o projections of a decoder: whole prompts, and the newest tokens over a paged
cache (`tensorpack_amd.cache.PagedCache`). No counterpart in the reference, whose layers end at the linear product.

Everything is computed by libmtc_hip.so (include/mtc_serve.h) in bf16 or f16 with fp32 sums and softmax, on the
current HIP stream; without a GPU these calls raise. Lengths and offsets stay on the device: no call
waits for the GPU, so a serving loop can capture them into a graph.
"""

import ctypes
import math
from typing import Optional

from . import _abi, _native
from .device import _need, current_stream_handle, prefill_workspace, require_gpu


def _dtype_code(dtype):
    import torch
    if dtype == torch.bfloat16:
        return _abi.MTC_DTYPE_BF16
    if dtype == torch.float16:
        return _abi.MTC_DTYPE_F16
    raise ValueError(f"attention takes bfloat16 or float16, got {dtype}")


def _kernel_heads(x):
    """x (rows, heads, dim) itself when the kernels can read it in place (unit stride along dim, the other strides
    multiples of 8 elements and rows that do not overlap, a 16-byte aligned start), else a contiguous copy."""
    r, h, u = x.stride()
    # (a stride along a length of one is never used)
    ok = (u == 1 and h % 8 == 0 and r % 8 == 0 and h >= 0 and x.shape[2] <= r < 1 << 24 and x.data_ptr() % 16 == 0)
    return x if ok else x.contiguous()


def _heads(x) -> "_abi.MtcHeads":
    return _abi.MtcHeads(x.data_ptr(), x.stride(0), x.stride(1))


def _int32(name, x, n, device):
    import torch
    _need(isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.dim() == 1 and x.is_contiguous()
          and x.device == device, f"{name} must be a contiguous 1-D int32 tensor on {device}")
    _need(n is None or x.shape[0] == n, f"{name} must hold {n} numbers, got {x.shape[0]}")
    return x.data_ptr()


def _scale(scale: Optional[float], dim: int) -> float:
    s = dim ** -0.5 if scale is None else float(scale)
    _need(math.isfinite(s) and s > 0, f"scale must be positive and finite, got {scale}")
    return s


def prompt_attention(q, k, v, cu_q, cu_k=None, *, causal: bool = True, scale: Optional[float] = None, out=None):
    """Attention over whole prompts packed one after another (mtc_prompt_attention).

    q (rows, heads, dim), k and v (keys, kv_heads, dim): bf16 or f16; strided views are read in place when their
    rows are 16-byte aligned. heads is a multiple of kv_heads, dim a multiple of 8 up to 128.
    cu_q, cu_k (sequences + 1) int32 on the device: sequence b owns rows cu_q[b]:cu_q[b+1] of q and
    cu_k[b]:cu_k[b+1] of k and v, from 0 to the end (cu_k None: cu_q). A sequence may have more keys than queries
    (the queries are then its last tokens), fewer, or none of either.
    causal: query t sees keys up to its own place; a query that sees none gives zeros.
    scale: of the scores; default dim ** -0.5. out: result tensor like q (rows outside every sequence keep what
    they held); default: a new contiguous tensor.
    """
    import torch
    dev = require_gpu(q.device)
    _need(q.dim() == 3 and k.dim() == 3 and v.dim() == 3, "q, k and v must be (tokens, heads, dim)")
    dt = _dtype_code(q.dtype)
    _need(k.dtype == q.dtype and v.dtype == q.dtype, f"q, k and v must share a dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    _need(k.device == dev and v.device == dev, f"q, k and v must be on {dev}")
    rows, heads, dim = q.shape
    _need(k.shape == v.shape and k.shape[2] == dim, f"k {tuple(k.shape)} and v {tuple(v.shape)} must be (keys, kv_heads, {dim})")
    kv_heads = k.shape[1]
    _need(kv_heads > 0 and heads > 0 and heads % kv_heads == 0, f"{heads} query heads over {kv_heads} K/V heads")
    _need(8 <= dim <= _abi.ATTN_MAX_DIM and dim % 8 == 0, f"dim must be a multiple of 8 from 8 to {_abi.ATTN_MAX_DIM}, got {dim}")
    scale = _scale(scale, dim)
    n = cu_q.shape[0] - 1 if cu_q.dim() == 1 else -1
    _need(n >= 0, "cu_q must hold sequences + 1 offsets")
    cq = _int32("cu_q", cu_q, None, dev)
    if cu_k is None:
        _need(k.shape[0] == rows, f"without cu_k, k and v hold one row per query: {k.shape[0]} != {rows}")
        ck = cq
    else:
        ck = _int32("cu_k", cu_k, n + 1, dev)
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=q.dtype, device=dev)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == dev and _kernel_heads(out) is out,
              f"out must be {tuple(q.shape)} {q.dtype} on {dev} with 16-byte aligned rows")
    q, k, v = _kernel_heads(q), _kernel_heads(k), _kernel_heads(v)
    lib = _native.hip_lib()
    args = _abi.MtcPromptArgs(_abi.ABI_VERSION, dt, n, heads, kv_heads, dim, rows, k.shape[0], int(causal), scale,
                              _heads(q), _heads(k), _heads(v), _heads(out), cq, ck)
    _abi.check(lib, "mtc_prompt_attention", lib.mtc_prompt_attention(ctypes.byref(args), current_stream_handle(dev)))
    return out


def cached_attention(q, cache, layer: int, seqs, *, q_lens=None, groups=None, prefix_lens=None,
                     scale: Optional[float] = None, out=None):
    """Attention of the newest tokens of each sequence over the cache, themselves included (mtc_cached_attention):
    call `cache.extend` and `cache.append` for them first.

    q (sequences, tokens, heads, dim), 1 to 16 tokens, in the cache's dtype; seqs (sequences) int32: their numbers in
    the cache. q_lens (sequences) int32: how many of the tokens count (the first ones of each row; the others
    give zeros); default all. Token t of sequence s sees the first lens[s] - q_lens + t + 1 tokens.
    groups (n + 1) int32 offsets into the batch and prefix_lens (n) int32: the sequences of a group hold the
    same pages for their first prefix_lens tokens (a `cache.fork` makes such sequences); these are read once
    and multiplied with all members' queries together. The result is that of a call without groups.
    scale, out: as for `prompt_attention`.
    """
    import torch
    dev = cache.device
    _need(q.dim() == 4 and q.device == dev, f"q must be (sequences, tokens, heads, dim) on {dev}")
    _need(q.dtype == cache.dtype, f"q must be {cache.dtype}, as the cache, got {q.dtype}")
    n, tokens, heads, dim = q.shape
    _need(dim == cache.head_dim, f"head size {dim}, the cache holds {cache.head_dim}")
    _need(heads > 0 and heads % cache.n_kv_heads == 0, f"{heads} query heads over {cache.n_kv_heads} K/V heads")
    _need(1 <= tokens <= _abi.CACHED_MAX_TOKENS, f"1 to {_abi.CACHED_MAX_TOKENS} tokens per sequence, got {tokens}")
    _need(n <= _abi.CACHED_MAX_SEQS, f"at most {_abi.CACHED_MAX_SEQS} sequences, got {n}")
    _need(0 <= layer < cache.n_layers, f"layer {layer} of {cache.n_layers}")
    _need((groups is None) == (prefix_lens is None), "groups and prefix_lens come together")
    scale = _scale(scale, dim)
    sp = _int32("seqs", seqs, n, dev)
    qp = None if q_lens is None else _int32("q_lens", q_lens, n, dev)
    gp = pp = None
    n_groups = 0
    if groups is not None:
        n_groups = prefix_lens.shape[0]
        pp, gp = _int32("prefix_lens", prefix_lens, None, dev), _int32("groups", groups, n_groups + 1, dev)
        _need(n_groups <= n, f"{n_groups} groups of {n} sequences")
    if out is None:
        out = torch.empty((n, tokens, heads, dim), dtype=q.dtype, device=dev)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == dev and out.is_contiguous()
              and out.data_ptr() % 16 == 0, f"out must be a contiguous {tuple(q.shape)} {q.dtype} tensor on {dev}")
    if n == 0:
        return out
    if tokens > 1 and q.stride(0) != tokens * q.stride(1):
        q = q.contiguous()
    # rows b * tokens + t
    qr = _kernel_heads(q.squeeze(1) if tokens == 1 else q.flatten(0, 1))
    lib = cache.lib
    args = _abi.MtcCachedArgs(_abi.ABI_VERSION, layer, n, tokens, heads, n_groups, scale, 0, _heads(qr),
                              _abi.MtcHeads(out.data_ptr(), heads * dim, dim), sp, qp, gp, pp)
    ref = ctypes.byref(args)
    need = int(lib.mtc_cached_attention_workspace_bytes(cache.desc_ref, ref))
    ws = prefill_workspace(dev, need) if need else None
    _abi.check(lib, "mtc_cached_attention",
               lib.mtc_cached_attention(cache.desc_ref, ref, ws.data_ptr() if need else None, need, current_stream_handle(dev)))
    return out
