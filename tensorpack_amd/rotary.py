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
from .attention import _aligned_rows, _apart, _copy, _heads, _int32
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
        if not math.isfinite(self.amplitude):
            raise ValueError(f"amplitude must be finite, got {amplitude}")
        f = rotary_frequencies(dim, base=base, factor=factor, original=original, ramp=ramp)
        if frequencies is not None:
            given = [float(x) for x in frequencies]
            if len(given) != len(f) or not all(math.isfinite(x) for x in given):
                raise ValueError(f"frequencies must be {len(f)} finite numbers, got {len(given)}")
            f = given
        self.frequencies = f
        turns = [round(Fraction(x) * 2 ** 63 / _PI) % 2 ** 64 for x in f]        # 2 ** 64 / (2 pi)
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64).to(self.device)


def apply_rotary(rotary: Rotary, q, k, positions, *, out=None):
    """(q', k'): q (rows, heads, dim) and k (rows, kv_heads, dim; or None) turned by their tokens' positions (mtc_rotary), in one launch.

    bf16, f16 or fp32; dim a multiple of 8 up to 1024; dims past rotary.dim are copied. positions (rows) int32 on the
    device, negative ones too. Strided views whose rows and heads are 16-byte aligned are read in place, others are copied.
    Angles, products and sums are fp32 or better, results rounded once. out: (q', k') to write to, which may be q and k themselves but
    share no other memory with them; default: new contiguous tensors."""
    import torch
    dev = rotary.device
    given = [x for x in (q, k) if x is not None]
    if q is None or any(x.dim() != 3 or x.shape[0] != q.shape[0] or x.shape[2] != q.shape[2] for x in given):
        raise ValueError(f"q and k must be (rows, heads, dim), got {[tuple(x.shape) for x in given]}")
    if any(x.device != dev or x.dtype != q.dtype for x in given):
        raise ValueError(f"q and k must share a dtype, on {dev}: {[(x.dtype, x.device) for x in given]}")
    code = {torch.float32: _abi.MTC_DTYPE_F32, torch.bfloat16: _abi.MTC_DTYPE_BF16, torch.float16: _abi.MTC_DTYPE_F16}.get(q.dtype)
    if code is None:
        raise ValueError(f"rotary positions take float32, bfloat16 or float16, got {q.dtype}")
    rows, heads, dim = q.shape
    if dim % 8 or not 8 <= dim <= _abi.ROTARY_MAX_DIM or rotary.dim > dim:
        raise ValueError(f"dim must be a multiple of 8 from {max(8, rotary.dim)} to {_abi.ROTARY_MAX_DIM}, got {dim}")
    p = _int32("positions", positions, rows, dev)
    if out is None:
        out = tuple(None if x is None else torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k))
    elif len(out) != 2 or (out[1] is None) != (k is None) or any(
            not (o.shape == x.shape and o.dtype == x.dtype and o.device == dev and _aligned_rows(o) and _apart(o)) for o, x in zip(out, given)):
        raise ValueError("out must be a pair of tensors like q and k with 16-byte aligned rows that do not overlap")
    ins = [x if _aligned_rows(x) else _copy(x) for x in given]
    none = _abi.MtcHeads(None, 0, 0)
    hq, hk = _heads(ins[0]), _heads(ins[1]) if k is not None else none
    args = _abi.MtcRotaryArgs(_abi.ABI_VERSION, code, rows, heads, 0 if k is None else k.shape[1], dim, rotary.dim, rotary.interleaved,
                              rotary.amplitude, 0, hq, hk, _heads(out[0]), _heads(out[1]) if k is not None else none, p,
                              rotary.turns.data_ptr())
    lib = _native.hip_lib()
    with on_device(dev.index):
        rc = lib.mtc_rotary(ctypes.byref(args), raw_stream(dev.index))
        if rc:
            _abi.check(lib, "mtc_rotary", rc)
    return tuple(out)
