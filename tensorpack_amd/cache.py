"""A paged K/V cache whose bookkeeping lives on the GPU (include/mtc_serve.h). No counterpart in the reference.

A page holds `page_size` tokens of every layer in one contiguous piece, so that copying one is one run of memory.
Sequences are rows of a table of page ids; a page may belong to several sequences (`fork`) and is copied when one
of them writes into it (`extend`). Free pages are those that no sequence holds; the lowest ids are given
out first, so every result is determined by the calls alone.

All calls are asynchronous on the current HIP stream and wait for nothing: lists of sequences, counts and lengths are
int32 tensors on the device. A bookkeeping call that cannot be done (no free page, a sequence twice, ...)
changes nothing and sets a bit in the cache's status; `check()` waits for the GPU and raises.
"""

import ctypes
from typing import Optional

from . import _abi, _native
from .attention import _copy, _dtype_code, _int32
from .device import _need, on_device, raw_stream, require_gpu

STATE_WORDS = 4


class CacheError(RuntimeError):
    """A bookkeeping call could not be done. `bits`: the status word (MTC_CACHE_*)."""

    def __init__(self, bits: int):
        super().__init__("; ".join(t for b, t in _abi.CACHE_STATUS.items() if bits & b) or f"status {bits}")
        self.bits = bits


class PagedCache:
    """n_pages pages of page_size tokens, n_layers layers of n_kv_heads heads of head_dim (a multiple of 8 up to 128),
    for up to max_seqs sequences of up to max_pages pages each. dtype: bfloat16 or float16. page_size: a power of
    two from 16 to 256.

    pool   (n_pages, n_layers, 2 (K, V), n_kv_heads, page_size, head_dim)
    table  (max_seqs, max_pages) int32 page ids, -1 past a sequence's last page
    lens   (max_seqs,) int32 tokens held
    refs   (n_pages,) int32 sequences that hold the page
    """

    def __init__(self, n_pages: int, n_layers: int, n_kv_heads: int, head_dim: int, *, max_seqs: int, max_pages: int,
                 page_size: int = 16, dtype=None, device=None, pool=None):
        import torch
        dtype = dtype or torch.bfloat16
        self.device = require_gpu(device if pool is None else pool.device)
        self.dtype = dtype
        self.n_pages, self.n_layers, self.n_kv_heads, self.head_dim = int(n_pages), int(n_layers), int(n_kv_heads), int(head_dim)
        self.page_size, self.max_seqs, self.max_pages = int(page_size), int(max_seqs), int(max_pages)
        code = _dtype_code(dtype)
        _need(min(self.n_pages, self.n_layers, self.n_kv_heads, self.max_seqs, self.max_pages) > 0, "sizes must be positive")
        _need(8 <= self.head_dim <= _abi.ATTN_MAX_DIM and self.head_dim % 8 == 0,
              f"head_dim must be a multiple of 8 from 8 to {_abi.ATTN_MAX_DIM}, got {head_dim}")
        _need(self.page_size in (16, 32, 64, 128, 256), f"page_size must be a power of two from 16 to 256, got {page_size}")
        _need(self.max_seqs <= _abi.CACHE_MAX_SLOTS, f"at most {_abi.CACHE_MAX_SLOTS} sequences, got {max_seqs}")
        shape = (self.n_pages, self.n_layers, 2, self.n_kv_heads, self.page_size, self.head_dim)
        if pool is None:
            pool = torch.empty(shape, dtype=dtype, device=self.device)
        _need(tuple(pool.shape) == shape and pool.dtype == dtype and pool.is_contiguous() and pool.data_ptr() % 16 == 0,
              f"pool must be a contiguous {shape} {dtype} tensor")
        self.pool = pool
        self.lib = _native.hip_lib()
        # one tensor for the bookkeeping, so that a snapshot is one copy
        entries, words = self.max_seqs * self.max_pages, (STATE_WORDS, self.max_seqs, self.n_pages)
        self.book = torch.zeros(sum(words) + entries, dtype=torch.int32, device=self.device)
        self.state, self.lens, self.refs, table = self.book.split([*words, entries])
        self.table = table.view(self.max_seqs, self.max_pages)
        self.table.fill_(-1)
        self.scratch = torch.empty(int(self.lib.mtc_cache_scratch_ints(self.n_pages, self.max_seqs)), dtype=torch.int32,
                                   device=self.device)
        self.desc = _abi.MtcCacheDesc(_abi.ABI_VERSION, code, self.n_pages, self.n_layers, self.n_kv_heads, self.head_dim,
                                      self.page_size, self.max_seqs, self.max_pages, 0, pool.data_ptr(), self.table.data_ptr(),
                                      self.lens.data_ptr(), self.refs.data_ptr(), self.state.data_ptr(), self.scratch.data_ptr())
        self.desc_ref = ctypes.byref(self.desc)
        _abi.check(self.lib, "mtc_check_cache_desc", self.lib.mtc_check_cache_desc(self.desc_ref))

    @classmethod
    def from_buffers(cls, pool, table, lens, refs) -> "PagedCache":
        """A cache over an existing pool (kept, not copied) with the given bookkeeping (copied)."""
        _need(pool.dim() == 6 and table.dim() == 2, "pool has six axes (see PagedCache), table two")
        self = cls(pool.shape[0], pool.shape[1], pool.shape[3], pool.shape[5], max_seqs=table.shape[0], max_pages=table.shape[1],
                   page_size=pool.shape[4], dtype=pool.dtype, pool=pool)
        for mine, given, name in ((self.table, table, "table"), (self.lens, lens, "lens"), (self.refs, refs, "refs")):
            _need(mine.shape == given.shape, f"{name} must be {tuple(mine.shape)}, got {tuple(given.shape)}")
            mine.copy_(given)
        return self

    # ---- bookkeeping ----------------------------------------------------------------
    def _call(self, name, *args):
        with on_device(self.device.index):
            rc = getattr(self.lib, name)(self.desc_ref, *args, raw_stream(self.device.index))
            if rc:
                _abi.check(self.lib, name, rc)

    def _list(self, name, x, n=None):
        if x.shape[0] > _abi.CACHED_MAX_SEQS:
            raise ValueError(f"{name}: at most {_abi.CACHED_MAX_SEQS} sequences a call")
        return _int32(name, x, n, self.device)

    def extend(self, seqs, counts) -> None:
        """Room for counts[i] more tokens of seqs[i]: lens grow, new pages are taken, a shared page that is
        partly filled is copied first. Write the tokens' K and V with `append`, layer by layer."""
        p = self._list("seqs", seqs)
        if seqs.shape[0] > self.max_seqs:
            raise ValueError(f"{seqs.shape[0]} sequences, the cache holds {self.max_seqs}")
        self._call("mtc_cache_extend", p, self._list("counts", counts, seqs.shape[0]), seqs.shape[0])

    def append(self, layer: int, k, v, seqs, cu) -> None:
        """Writes K and V (rows, n_kv_heads, head_dim; the cache's dtype, or fp32 to be rounded) of the newest tokens:
        rows cu[i]:cu[i+1] are the last tokens of seqs[i]. cu: (sequences + 1) int32 offsets from 0."""
        import torch
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        if k.dim() != 3 or k.shape != v.shape or k.shape[1] != self.n_kv_heads or k.shape[2] != self.head_dim:
            raise ValueError(f"k and v must be (rows, {self.n_kv_heads}, {self.head_dim}), got {tuple(k.shape)}, {tuple(v.shape)}")
        if not (k.dtype == v.dtype and k.dtype in (self.dtype, torch.float32) and k.device == self.device == v.device):
            raise ValueError(f"k and v must be {self.dtype} or float32 on {self.device}")
        p = self._list("seqs", seqs)
        c = _int32("cu", cu, seqs.shape[0] + 1, self.device)
        mask = 16 // k.element_size() - 1                        # rows of 16-byte pieces are read in place, others copied
        k, v = (x if x.stride(2) == 1 and not (x.stride(0) | x.stride(1)) & mask and not x.data_ptr() & 15 else _copy(x)
                for x in (k, v))
        hk, hv = (_abi.MtcHeads(x.data_ptr(), x.stride(0), x.stride(1)) for x in (k, v))
        code = _abi.MTC_DTYPE_F32 if k.dtype == torch.float32 else self.desc.dtype
        self._call("mtc_cache_append", layer, ctypes.byref(hk), ctypes.byref(hv), code, k.shape[0], p, c, seqs.shape[0])

    def fork(self, src, dst) -> None:
        """dst[i] (empty) becomes a second holder of everything src[i] holds. src may name a sequence several times."""
        p = self._list("src", src)
        self._call("mtc_cache_fork", p, self._list("dst", dst, src.shape[0]), src.shape[0])

    def truncate(self, seqs, new_lens) -> None:
        """seqs[i] keeps its first new_lens[i] tokens; pages that nobody holds any more become free."""
        p = self._list("seqs", seqs)
        self._call("mtc_cache_truncate", p, self._list("new_lens", new_lens, seqs.shape[0]), seqs.shape[0])

    def free(self, seqs) -> None:
        """seqs hold nothing any more."""
        self._call("mtc_cache_truncate", self._list("seqs", seqs), None, seqs.shape[0])

    def compact(self) -> None:
        """Moves pages so that those in use have the lowest ids (`pool` past them can then be cut off or given away)."""
        self._call("mtc_cache_compact")

    def copy_pages(self, src, dst, source: Optional["PagedCache"] = None) -> None:
        """Page dst[i] becomes a copy of page src[i] of `source` (a cache of the same geometry; default: this one).
        dst are distinct and none of them is also a src of this cache. Ids out of range copy nothing."""
        source = source or self
        _need(source.device == self.device and source.dtype == self.dtype and source.pool.shape[1:] == self.pool.shape[1:],
              "source must have the same page geometry and dtype, on the same device")
        p, n = _int32("src", src, None, self.device), src.shape[0]
        self._call("mtc_cache_copy_pages", source.pool.data_ptr(), source.n_pages, p, _int32("dst", dst, n, self.device), n)

    def snapshot(self):
        """The bookkeeping as it is now (not the pages' contents), for `restore`."""
        return self.book.clone()

    def restore(self, snapshot) -> None:
        """Puts the bookkeeping back, but for the status: `check()` still raises, once, for a call since the last check.
        Pages written or moved since hold what was written."""
        _need(snapshot.shape == self.book.shape and snapshot.dtype == self.book.dtype, "not a snapshot of this cache")
        self.book[1:].copy_(snapshot[1:])

    def check(self) -> None:
        """Waits for the GPU; raises CacheError if a call since the last check could not be done."""
        bits = int(self.state[0].item())
        if bits:
            self.state[0] = 0
            raise CacheError(bits)

    @property
    def free_pages(self) -> int:
        """Pages that no sequence holds (waits for the GPU)."""
        return int((self.refs == 0).sum().item())
