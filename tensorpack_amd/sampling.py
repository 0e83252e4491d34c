"""Verification of drafted tokens (include/mtc_serve.h). No counterpart in the reference.

A small model drafts a few tokens per sequence; the large one scores them in one pass (at 2 to 16 rows the packed
matmul reads its weights once, as for one) and keeps a run of them so that the tokens have the large
model's distribution.
"""

import ctypes

from . import _abi, _native
from .device import _need, current_stream_handle, prefill_workspace, require_gpu


def verify_drafts(drafts, p, q, u, noise, *, n_drafts=None):
    """(tokens, accepted) of a batch of drafts (mtc_verify_drafts).

    drafts (B, K) int32 or int64, drawn from q; p (B, K + 1, V): the target's probabilities after each draft; q
    (B, K, V): the draft model's; both fp32, bf16 or f16, unit stride along V. u (B, K) fp32 uniform in [0, 1);
    noise (B, V) fp32: 1 / Exp(1) draws. n_drafts (B) int32: drafts per sequence (default K).
    Draft j is accepted while u[j] * q[j, x] < p[j, x]. The next token is the first index of the largest w * noise over
    w > 0 (distributed as w / sum(w)), with w = max(p - q, 0) at the first rejected draft (p where that is 0
    everywhere), or p after the last accepted one; -1 if no w > 0.
    tokens (B, K + 1) in drafts' dtype: the accepted drafts, the next token, then -1. accepted (B) int32.
    """
    import torch
    dev = require_gpu(p.device)
    _need(drafts.dim() == 2 and p.dim() == 3 and q.dim() == 3 and u.dim() == 2 and noise.dim() == 2,
          "drafts (B, K), p (B, K + 1, V), q (B, K, V), u (B, K), noise (B, V)")
    B, K = drafts.shape
    V = p.shape[2]
    _need(tuple(p.shape) == (B, K + 1, V) and tuple(q.shape) == (B, K, V) and tuple(u.shape) == (B, K)
          and tuple(noise.shape) == (B, V) and V > 0,
          f"shapes do not fit: drafts {tuple(drafts.shape)}, p {tuple(p.shape)}, q {tuple(q.shape)}, u {tuple(u.shape)}, noise {tuple(noise.shape)}")
    codes = {torch.float32: _abi.MTC_DTYPE_F32, torch.bfloat16: _abi.MTC_DTYPE_BF16, torch.float16: _abi.MTC_DTYPE_F16}
    _need(p.dtype in codes and q.dtype == p.dtype, f"p and q must share a dtype of fp32, bf16 or f16, got {p.dtype}, {q.dtype}")
    _need(drafts.dtype in (torch.int32, torch.int64), f"drafts must be int32 or int64, got {drafts.dtype}")
    _need(u.dtype == torch.float32 and noise.dtype == torch.float32, "u and noise must be fp32")
    _need(all(t.device == dev for t in (drafts, q, u, noise)), f"all inputs must be on {dev}")
    _need(K <= 64, f"at most 64 drafts, got {K}")
    _need(B <= 65535, f"at most 65535 sequences, got {B}")
    unit = lambda t: t if t.stride(-1) == 1 else t.contiguous()
    drafts, p, q, u, noise = (unit(t) for t in (drafts, p, q, u, noise))
    np_ = None
    if n_drafts is not None:
        _need(n_drafts.dtype == torch.int32 and tuple(n_drafts.shape) == (B,) and n_drafts.is_contiguous()
              and n_drafts.device == dev, f"n_drafts must be ({B},) int32 on {dev}")
        np_ = n_drafts.data_ptr()
    tokens = torch.empty((B, K + 1), dtype=drafts.dtype, device=dev)
    accepted = torch.empty((B,), dtype=torch.int32, device=dev)
    if B == 0:
        return tokens, accepted
    lib = _native.hip_lib()
    two = ctypes.c_int64 * 2
    args = _abi.MtcVerifyArgs(_abi.ABI_VERSION, codes[p.dtype], drafts.element_size(), B, K, V, p.data_ptr(),
                              two(p.stride(0), p.stride(1)), q.data_ptr(), two(q.stride(0), q.stride(1)), u.data_ptr(), u.stride(0),
                              noise.data_ptr(), noise.stride(0), drafts.data_ptr(), drafts.stride(0), np_, tokens.data_ptr(),
                              accepted.data_ptr())
    ref = ctypes.byref(args)
    need = int(lib.mtc_verify_workspace_bytes(ref))
    ws = prefill_workspace(dev, need)
    _abi.check(lib, "mtc_verify_drafts", lib.mtc_verify_drafts(ref, ws.data_ptr(), need, current_stream_handle(dev)))
    return tokens, accepted
