"""Attention between the q/k/v and o projections of a decoder: whole prompts, and the newest tokens over a paged
cache (`tensorpack_amd.cache.PagedCache`). No counterpart in the reference, whose layers end at the linear product.

Everything is computed by libmtc_hip.so (include/mtc_serve.h) in bf16 or f16 with fp32 sums and softmax, on the
current HIP stream; without a GPU these calls raise. Lengths and offsets stay on the device: no call
waits for the GPU, so a serving loop can capture them into a graph.
"""

import ctypes
import functools
from typing import Optional

from . import _abi, _native
from .device import on_device, raw_stream, require_gpu, stream_workspace


def _dtype_code(dtype):
    import torch
    if dtype == torch.bfloat16:
        return _abi.MTC_DTYPE_BF16
    if dtype == torch.float16:
        return _abi.MTC_DTYPE_F16
    raise ValueError(f"attention takes bfloat16 or float16, got {dtype}")


@functools.lru_cache(maxsize=None)
def _value_code(dtype):
    """MTC_DTYPE_* of float32, bfloat16 or float16, None for others."""
    import torch
    return {torch.float32: _abi.MTC_DTYPE_F32, torch.bfloat16: _abi.MTC_DTYPE_BF16, torch.float16: _abi.MTC_DTYPE_F16}.get(dtype)


def _in_place(x) -> bool:
    """The kernels can take x (rows, heads, dim) where it is: unit stride along dim, the other strides multiples of 8
    elements, rows that do not overlap, a 16-byte aligned start."""
    r, h, u = x.stride()
    return u == 1 and not (h | r) & 7 and x.shape[2] <= r < 1 << 24 and not x.data_ptr() & 15


def _aligned_rows(x) -> bool:
    """x (rows, heads, dim) of any type: unit stride along dim, rows and heads that start at multiples of 16 bytes."""
    r, h, u = x.stride()
    return u == 1 and not (h | r) * x.element_size() & 15 and not x.data_ptr() & 15


def _apart(x) -> bool:
    """No two elements of x (rows, heads, dim) share memory."""
    end = x.shape[2]
    for stride, size in sorted((s, n) for s, n in zip(x.stride()[:2], x.shape[:2]) if n > 1):
        if stride < end:
            return False
        end += stride * (size - 1)
    return True


def _meet(a, a_shape, b, b_shape, size: int) -> bool:
    """Two views of (rows, heads, dim) elements of `size` bytes, each given as (address, row stride, head stride) with unit stride along
    the same dim, share memory. Addresses are multiples of `size`."""
    (at, r, h), (rows, heads, dim) = a, a_shape
    (at2, r2, h2), (rows2, heads2, _) = b, b_shape
    if not (rows and heads and rows2 and heads2):
        return False
    apart, block, block2 = (at2 - at) // size, (heads - 1) * h + dim, (heads2 - 1) * h2 + dim
    if apart >= (rows - 1) * r + block or -apart >= (rows2 - 1) * r2 + block2:
        return False
    if r == r2 and r and block <= apart % r <= r - block2:         # parts of the rows of one buffer
        return False
    import torch
    first = (torch.arange(rows)[:, None] * r + torch.arange(heads) * h).flatten().sort().values
    second = (torch.arange(rows2)[:, None] * r2 + torch.arange(heads2) * h2).flatten() + apart
    after = torch.searchsorted(first, second, right=True)
    low = second - first[(after - 1).clamp(min=0)] < dim
    high = first[after.clamp(max=first.numel() - 1)] - second < dim
    return bool(((after > 0) & low | (after < first.numel()) & high).any())


def _copy(x):
    """A contiguous copy in memory of its own. (contiguous() returns x itself where only its start or the stride of an
    axis of size 1 is in the way.)"""
    import torch
    return x.clone(memory_format=torch.contiguous_format)


def _kernel_heads(x):
    return x if _in_place(x) else _copy(x)


def _heads(x) -> "_abi.MtcHeads":
    return _abi.MtcHeads(x.data_ptr(), x.stride(0), x.stride(1))


def _int32(name, x, n, device):
    """Address of a list of n (None: any number of) int32 on the device."""
    import torch
    if not (isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.dim() == 1 and x.is_contiguous() and x.device == device):
        raise ValueError(f"{name} must be a contiguous 1-D int32 tensor on {device}")
    if n is not None and x.shape[0] != n:
        raise ValueError(f"{name} must hold {n} numbers, got {x.shape[0]}")
    return x.data_ptr()


_F32_MAX = (2 - 2 ** -23) * 2.0 ** 127


def _scale(scale: Optional[float], dim: int) -> float:
    if scale is None:
        return dim ** -0.5
    if not 0 < scale <= _F32_MAX:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return float(scale)


def prompt_attention(q, k, v, cu_q, cu_k=None, *, causal: bool = True, scale: Optional[float] = None, out=None):
    """Attention over whole prompts packed one after another (mtc_prompt_attention).

    q (rows, heads, dim), k and v (keys, kv_heads, dim): bf16 or f16; strided views are read in place when their
    rows are 16-byte aligned, others are copied. heads is a multiple of kv_heads, dim a multiple of 8 up to 128.
    cu_q, cu_k (sequences + 1) int32 on the device: sequence b owns rows cu_q[b]:cu_q[b+1] of q and
    cu_k[b]:cu_k[b+1] of k and v, from 0 to the end (cu_k None: cu_q). A sequence may have more keys than queries
    (the queries are then its last tokens), fewer, or none of either.
    causal: query t sees keys up to its own place; a query that sees none gives zeros.
    scale: of the scores; default dim ** -0.5. out: result tensor like q (rows outside every sequence keep what
    they held); it may be q itself, but shares no other memory with q, k or v; default: a new contiguous tensor.
    """
    import torch
    dev = q.device if q.is_cuda else require_gpu(q.device)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"q, k and v must be (tokens, heads, dim), k and v alike: {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    dt = _dtype_code(q.dtype)
    if not (k.dtype == q.dtype == v.dtype and k.device == dev == v.device):
        raise ValueError(f"q, k and v must share dtype and device, got {q.dtype}, {k.dtype}, {v.dtype} on {dev}, {k.device}, {v.device}")
    rows, heads, dim = q.shape
    keys, kv_heads, k_dim = k.shape
    if k_dim != dim or kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads of {dim} over {kv_heads} K/V heads of {k_dim}")
    if dim < 8 or dim > _abi.ATTN_MAX_DIM or dim % 8:
        raise ValueError(f"dim must be a multiple of 8 from 8 to {_abi.ATTN_MAX_DIM}, got {dim}")
    scale = _scale(scale, dim)
    cq = _int32("cu_q", cu_q, None, dev)
    n = cu_q.shape[0] - 1
    if n < 0:
        raise ValueError("cu_q must hold sequences + 1 offsets")
    if cu_k is not None:
        ck = _int32("cu_k", cu_k, n + 1, dev)
    elif keys == rows:
        ck = cq
    else:
        raise ValueError(f"without cu_k, k and v hold one row per query: {keys} != {rows}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif not (out.shape == q.shape and out.dtype == q.dtype and out.device == dev and _in_place(out)):
        raise ValueError(f"out must be {tuple(q.shape)} {q.dtype} on {dev} with 16-byte aligned rows")
    elif rows and keys and out.data_ptr() in (k.data_ptr(), v.data_ptr()):
        raise ValueError("out is k or v, which other rows still read")
    lib = _native.hip_lib()
    q, k, v = _kernel_heads(q), _kernel_heads(k), _kernel_heads(v)
    args = _abi.MtcPromptArgs(_abi.ABI_VERSION, dt, n, heads, kv_heads, dim, rows, keys, causal, scale,
                              _heads(q), _heads(k), _heads(v), _heads(out), cq, ck)
    ref, stream = ctypes.byref(args), raw_stream(dev.index)
    need = lib.mtc_prompt_attention_workspace_bytes(ref)
    with on_device(dev.index):
        ws = stream_workspace(dev.index, stream, need) if need else None
        rc = lib.mtc_prompt_attention(ref, ws.data_ptr() if need else None, need, stream)
        if rc:
            _abi.check(lib, "mtc_prompt_attention", rc)
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
    if q.dim() != 4 or q.device != dev or q.dtype != cache.dtype:
        raise ValueError(f"q must be (sequences, tokens, heads, dim) {cache.dtype} on {dev}, got {tuple(q.shape)} {q.dtype} on {q.device}")
    n, tokens, heads, dim = q.shape
    if dim != cache.head_dim or heads < 1 or heads % cache.n_kv_heads:
        raise ValueError(f"{heads} query heads of {dim} over a cache of {cache.n_kv_heads} heads of {cache.head_dim}")
    if not 1 <= tokens <= _abi.CACHED_MAX_TOKENS:
        raise ValueError(f"1 to {_abi.CACHED_MAX_TOKENS} tokens per sequence, got {tokens}")
    if n > _abi.CACHED_MAX_SEQS:
        raise ValueError(f"at most {_abi.CACHED_MAX_SEQS} sequences, got {n}")
    if not 0 <= layer < cache.n_layers:
        raise ValueError(f"layer {layer} of {cache.n_layers}")
    scale = _scale(scale, dim)
    sp = _int32("seqs", seqs, n, dev)
    qp = None if q_lens is None else _int32("q_lens", q_lens, n, dev)
    gp = pp = None
    n_groups = 0
    if (groups is None) != (prefix_lens is None):
        raise ValueError("groups and prefix_lens come together")
    if groups is not None:
        n_groups = prefix_lens.shape[0]
        pp, gp = _int32("prefix_lens", prefix_lens, None, dev), _int32("groups", groups, n_groups + 1, dev)
        if n_groups > n:
            raise ValueError(f"{n_groups} groups of {n} sequences")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif not (out.shape == q.shape and out.dtype == q.dtype and out.device == dev and out.is_contiguous() and out.data_ptr() % 16 == 0):
        raise ValueError(f"out must be a contiguous {tuple(q.shape)} {q.dtype} tensor on {dev}")
    if n == 0:
        return out
    # rows b * tokens + t
    if tokens > 1 and q.stride(0) != tokens * q.stride(1):
        q = q.contiguous()
    row, head, unit = q.stride(0) if tokens == 1 else q.stride(1), q.stride(2), q.stride(3)
    if unit != 1 or (row | head) & 7 or not dim <= row < 1 << 24 or q.data_ptr() & 15:
        q = _copy(q)
        row, head = heads * dim, dim
    lib = cache.lib
    args = _abi.MtcCachedArgs.from_buffer_copy(_abi.CACHED_PACK(
        _abi.ABI_VERSION, layer, n, tokens, heads, n_groups, scale, 0, q.data_ptr(), row, head, out.data_ptr(), heads * dim, dim, sp,
        qp or 0, gp or 0, pp or 0))
    ref, stream = ctypes.byref(args), raw_stream(dev.index)
    need = lib.mtc_cached_attention_workspace_bytes(cache.desc_ref, ref)
    with on_device(dev.index):
        ws = stream_workspace(dev.index, stream, need) if need else None
        rc = lib.mtc_cached_attention(cache.desc_ref, ref, ws.data_ptr() if need else None, need, stream)
        if rc:
            _abi.check(lib, "mtc_cached_attention", rc)
    return out
