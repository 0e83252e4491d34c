"""Verification of drafted tokens, and a step of beam search (include/mtc_serve.h). No counterpart in the reference.

A small model drafts a few tokens per sequence; the large one scores them in one pass (at 2 to 16 rows the packed
matmul reads its weights once, as for one) and keeps a run of them so that the tokens have the large
model's distribution.
"""

import ctypes
from typing import Optional

from . import _abi, _native
from .attention import _value_code
from .device import on_device, raw_stream, require_gpu, stream_workspace


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
    dev = p.device if p.is_cuda else require_gpu(p.device)
    if drafts.dim() != 2 or p.dim() != 3:
        raise ValueError("drafts (B, K), p (B, K + 1, V), q (B, K, V), u (B, K), noise (B, V)")
    (B, K), V = drafts.shape, p.shape[2]
    if p.shape != (B, K + 1, V) or q.shape != (B, K, V) or u.shape != (B, K) or noise.shape != (B, V) or V < 1:
        raise ValueError(f"shapes do not fit: drafts {tuple(drafts.shape)}, p {tuple(p.shape)}, q {tuple(q.shape)}, u {tuple(u.shape)}, "
                         f"noise {tuple(noise.shape)}")
    code = {torch.float32: _abi.MTC_DTYPE_F32, torch.bfloat16: _abi.MTC_DTYPE_BF16, torch.float16: _abi.MTC_DTYPE_F16}.get(p.dtype)
    if code is None or q.dtype != p.dtype:
        raise ValueError(f"p and q must share a dtype of fp32, bf16 or f16, got {p.dtype}, {q.dtype}")
    if drafts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"drafts must be int32 or int64, got {drafts.dtype}")
    if u.dtype != torch.float32 or noise.dtype != torch.float32:
        raise ValueError("u and noise must be fp32")
    if not (drafts.device == dev == q.device and u.device == dev == noise.device):
        raise ValueError(f"all inputs must be on {dev}")
    if K > 64 or B > 65535:
        raise ValueError(f"at most 65535 sequences of 64 drafts, got {B} of {K}")
    np_ = None
    if n_drafts is not None:
        if not (n_drafts.dtype == torch.int32 and n_drafts.shape == (B,) and n_drafts.is_contiguous() and n_drafts.device == dev):
            raise ValueError(f"n_drafts must be ({B},) int32 on {dev}")
        np_ = n_drafts.data_ptr()
    tokens = torch.empty((B, K + 1), dtype=drafts.dtype, device=dev)
    accepted = torch.empty((B,), dtype=torch.int32, device=dev)
    if B == 0:
        return tokens, accepted
    drafts, p, q, u, noise = (t if t.stride(-1) == 1 else t.contiguous() for t in (drafts, p, q, u, noise))
    lib = _native.hip_lib()
    args = _abi.MtcVerifyArgs(_abi.ABI_VERSION, code, drafts.element_size(), B, K, V, p.data_ptr(), p.stride()[:2], q.data_ptr(),
                              q.stride()[:2], u.data_ptr(), u.stride(0), noise.data_ptr(), noise.stride(0), drafts.data_ptr(),
                              drafts.stride(0), np_, tokens.data_ptr(), accepted.data_ptr())
    ref, stream = ctypes.byref(args), raw_stream(dev.index)
    need = lib.mtc_verify_workspace_bytes(ref)
    with on_device(dev.index):
        ws = stream_workspace(dev.index, stream, need)
        rc = lib.mtc_verify_drafts(ref, ws.data_ptr(), need, stream)
        if rc:
            _abi.check(lib, "mtc_verify_drafts", rc)
    return tokens, accepted


def beam_select(logits, scores, *, n: Optional[int] = None, done=None, pad: int = 0):
    """(scores, tokens, parents), each (B, n): the n best continuations of each prompt's W beams (mtc_beam_select).

    logits (B, W, V) fp32, bf16 or f16, unit stride along V (else copied), up to 65535 rows; scores (B, W) fp32: the beams' log
    probabilities so far. n: default W, at most 64, as W. A continuation's score is scores[b, w] + log_softmax(logits[b, w])[v]; the best
    come first, equal ones in the order of w * V + v. A log sum is off by less than 2.7e-6 (V up to 2 ** 20; usually a tenth of that): of two beams'
    continuations that lie closer, either may come first. done (B, W) bool: beams that have ended; such a beam stands as one candidate
    with its score as it is and the token `pad`. Scores of -inf are no candidates (give all beams but one -inf at the first step, or tokens
    that must not come a logit of -inf).
    scores fp32, tokens int32, parents int32: the row b * W + w of the beam that goes on, as it stands in `logits.flatten(0, 1)`, and in the
    list for `PagedCache.reorder` where n = W. Where there are fewer candidates than n: -inf, -1 and some row of the prompt.
    """
    import torch
    dev = logits.device if logits.is_cuda else require_gpu(logits.device)
    if logits.dim() != 3 or scores.shape != logits.shape[:2]:
        raise ValueError(f"logits (B, W, V) and scores (B, W), got {tuple(logits.shape)}, {tuple(scores.shape)}")
    B, W, V = logits.shape
    n = W if n is None else n
    code = _value_code(logits.dtype)
    if code is None or scores.dtype != torch.float32:
        raise ValueError(f"logits must be fp32, bf16 or f16, scores fp32, got {logits.dtype}, {scores.dtype}")
    if not 1 <= W <= _abi.BEAM_MAX or not 1 <= n <= _abi.BEAM_MAX or V < 1:
        raise ValueError(f"1 to {_abi.BEAM_MAX} beams and picks over a vocabulary, got {W}, {n}, {V}")
    if scores.device != dev or (done is not None and not (done.dtype == torch.bool and done.shape == scores.shape and done.device == dev)):
        raise ValueError(f"scores must be on {dev}, and done {tuple(scores.shape)} bool there")
    if not -1 << 31 <= pad < 1 << 31:
        raise ValueError(f"pad must fit 32 bits, got {pad}")
    best, tokens, parents = torch.empty((3, B, n), dtype=torch.int32, device=dev).unbind(0)
    best = best.view(torch.float32)
    if B == 0:
        return best, tokens, parents
    if logits.stride(2) != 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    if done is not None:
        done = done.contiguous()
    lib = _native.hip_lib()
    args = _abi.MtcBeamArgs.from_buffer_copy(_abi.BEAM_PACK(
        _abi.ABI_VERSION, code, B, W, V, n, pad, 0, logits.data_ptr(), logits.stride(0), logits.stride(1), scores.data_ptr(),
        0 if done is None else done.data_ptr(), best.data_ptr(), tokens.data_ptr(), parents.data_ptr()))
    ref, stream = ctypes.byref(args), raw_stream(dev.index)
    need = lib.mtc_beam_workspace_bytes(ref)
    with on_device(dev.index):
        ws = stream_workspace(dev.index, stream, need)
        rc = lib.mtc_beam_select(ref, ws.data_ptr(), need, stream)
        if rc:
            _abi.check(lib, "mtc_beam_select", rc)
    return best, tokens, parents
