"""Rotary positions for the queries and keys of a decoder (include/mtc_serve.h). No counterpart in the reference, whose
layers end at the linear product.

Pair i of a head's first `dim` dims is turned by its token's position times f_i. The turn is computed in 64-bit
fixed point, so it is as exact at position 2 000 000 000 as at 1; nothing is kept but the frequencies.
"""

import ctypes
import math
from fractions import Fraction
from typing import Optional, Sequence

from . import _abi, _native
from .attention import _F32_MAX, _aligned_rows, _apart, _copy, _int32, _meet, _value_code
from .device import on_device, raw_stream, require_gpu

_PI = Fraction(3141592653589793238462643383279502884197169399375105820974944592307816406286, 10 ** 75)


def rotary_frequencies(dim: int, *, base: float = 10000.0, factor: float = 1.0, original: Optional[int] = None, ramp=(1.0, 4.0)):
    """f_i = base ** (-2 i / dim), i < dim / 2, in radians per token. factor > 1 stretches the context:
    f_i / factor, or with `original` (the length of the context before) blended by how often a pair turns within it,
    r_i = original f_i / 2 pi: pairs of ramp[1] turns or more keep f_i, those of ramp[0] or fewer get f_i / factor,
    those between a mixture, linear in r_i."""
    if dim < 2 or dim % 2:
        raise ValueError(f"an even count of dims is turned, got {dim}")
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor >= 1):
        raise ValueError(f"base must be positive and finite, factor 1 or more, got {base}, {factor}")
    if original is not None and not (original > 0 and 0 <= ramp[0] < ramp[1]):
        raise ValueError(f"original must be positive, ramp two rising numbers, got {original}, {ramp}")
    out = []
    for i in range(dim // 2):
        f = base ** (-2.0 * i / dim)
        keep = 0.0
        if original is not None:
            keep = min(1.0, max(0.0, (original * f / (2.0 * math.pi) - ramp[0]) / (ramp[1] - ramp[0])))
        out.append(f * (keep + (1.0 - keep) / factor))
    return out


class Rotary:
    """What `apply_rotary` turns by: the first `dim` (even) dims of a head, as pairs (i, i + dim / 2), or (2 i, 2 i + 1) with
    `interleaved`. frequencies: dim / 2 numbers in radians per token, the first pair's first; default: rotary_frequencies of the other
    arguments. amplitude: a factor on the turned dims (some stretched contexts use one)."""

    def __init__(self, dim: int, *, base: float = 10000.0, interleaved: bool = False, factor: float = 1.0, original: Optional[int] = None,
                 ramp=(1.0, 4.0), amplitude: float = 1.0, frequencies: Optional[Sequence[float]] = None, device=None):
        import torch
        self.device = require_gpu(device)
        self.dim, self.interleaved, self.amplitude = int(dim), bool(interleaved), float(amplitude)
        if not abs(self.amplitude) <= _F32_MAX:
            raise ValueError(f"amplitude must be a finite fp32 number, got {amplitude}")
        f = rotary_frequencies(dim, base=base, factor=factor, original=original, ramp=ramp)
        if frequencies is not None:
            given = [float(x) for x in frequencies]
            if len(given) != len(f) or not all(math.isfinite(x) for x in given):
                raise ValueError(f"frequencies must be {len(f)} finite numbers, got {len(given)}")
            f = given
        self.frequencies = f
        turns = [round(Fraction(x) * 2 ** 63 / _PI) % 2 ** 64 for x in f]        # 2 ** 64 / (2 pi)
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64).to(self.device)
        self.turns_at = self.turns.data_ptr()


_NONE = (0, 0, 0)


def _view(x):
    r, h, _ = x.stride()
    return x.data_ptr(), r, h


def _readable(x, mask):
    """x, or a copy that the kernel can read, and its address and strides."""
    (r, h, u), at = x.stride(), x.data_ptr()
    if u == 1 and not (r | h) & mask and not at & 15:
        return x, (at, r, h)
    x = _copy(x)
    return x, _view(x)


def _like(out, x) -> bool:
    return out.shape == x.shape and out.dtype == x.dtype and out.device == x.device and _aligned_rows(out) and _apart(out)


def _clash(hq, ho, heads, hk, ok, kv_heads, rows, dim, size) -> bool:
    """A result (ho, ok: address, strides) shares memory with anything but its own input, element by element."""
    q, k = (rows, heads, dim), (rows, kv_heads, dim)
    own = lambda a, b, n: a[0] == b[0] and (rows < 2 or a[1] == b[1]) and (n < 2 or a[2] == b[2])
    q_own, k_own = own(hq, ho, heads), own(hk, ok, kv_heads)         # an input in the place of its result: one pair less
    return (not q_own and _meet(ho, q, hq, q, size)) or (not k_own and _meet(ok, k, hk, k, size)) or _meet(ho, q, ok, k, size) or \
        (not k_own and _meet(ho, q, hk, k, size)) or (not q_own and _meet(ok, k, hq, q, size))


def apply_rotary(rotary: Rotary, q, k, positions, *, out=None):
    """(q', k'): q (rows, heads, dim) and k (rows, kv_heads, dim; or None) turned by their tokens' positions (mtc_rotary), in one launch.

    bf16, f16 or fp32; dim a multiple of 8 up to 1024; dims past rotary.dim are copied. positions (rows) int32 on the
    device, negative ones too. Strided views whose rows and heads are 16-byte aligned are read in place, others are copied.
    Angles, products and sums are fp32 or better, results rounded once. out: (q', k') to write to, which may be q and k themselves (the
    same elements in the same places) but share no other memory with them or with each other; default: new contiguous tensors."""
    import torch
    dev = rotary.device
    if q.dim() != 3 or q.device != dev:
        raise ValueError(f"q must be (rows, heads, dim) on {dev}, got {tuple(q.shape)} on {q.device}")
    rows, heads, dim = q.shape
    dtype = q.dtype
    kv_heads = 0
    if k is not None:
        if k.dim() != 3 or k.dtype != dtype or k.device != dev:
            raise ValueError(f"k must be ({rows}, kv_heads, {dim}) {dtype} on {dev}, got {tuple(k.shape)} {k.dtype} on {k.device}")
        k_rows, kv_heads, k_dim = k.shape
        if k_rows != rows or k_dim != dim:
            raise ValueError(f"k must be ({rows}, kv_heads, {dim}), got {tuple(k.shape)}")
    code = _value_code(dtype)
    if code is None:
        raise ValueError(f"rotary positions take float32, bfloat16 or float16, got {dtype}")
    if dim % 8 or not 8 <= dim <= _abi.ROTARY_MAX_DIM or rotary.dim > dim:
        raise ValueError(f"dim must be a multiple of 8 from {max(8, rotary.dim)} to {_abi.ROTARY_MAX_DIM}, got {dim}")
    p = _int32("positions", positions, rows, dev)
    mask = 15 // dtype.itemsize                              # strides of rows of 16-byte pieces have none of these bits
    q, hq = _readable(q, mask)
    hk = ok = _NONE
    if k is not None:
        k, hk = _readable(k, mask)
    if out is None:
        new = torch.contiguous_format
        oq = torch.empty_like(q, memory_format=new)
        ho = oq.data_ptr(), heads * dim, dim
        out = oq, None
        if k is not None:
            out = oq, torch.empty_like(k, memory_format=new)
            ok = out[1].data_ptr(), kv_heads * dim, dim
    else:
        out = tuple(out)
        if len(out) != 2 or not _like(out[0], q) or (k is None) != (out[1] is None) or not (k is None or _like(out[1], k)):
            raise ValueError("out must be a pair of tensors like q and k with 16-byte aligned rows that do not overlap")
        ho = _view(out[0])
        if k is not None:
            ok = _view(out[1])
        if _clash(hq, ho, heads, hk, ok, kv_heads, rows, dim, dtype.itemsize):
            raise ValueError("the results share memory with each other, with the other one's input, or with their own at other places")
    args = _abi.MtcRotaryArgs.from_buffer_copy(_abi.ROTARY_PACK(
        _abi.ABI_VERSION, code, rows, heads, kv_heads, dim, rotary.dim, rotary.interleaved, rotary.amplitude, 0, *hq, *hk, *ho, *ok, p,
        rotary.turns_at))
    lib = _native.hip_lib()
    with on_device(dev.index):
        rc = lib.mtc_rotary(ctypes.byref(args), raw_stream(dev.index))
        if rc:
            _abi.check(lib, "mtc_rotary", rc)
    return out
