"""Verification of drafted tokens (speculative decoding).

``verify_draft`` decides, on the device and without a host sync, how many of
each sequence's drafted tokens the target model keeps and which token follows
them (``akv_verify_draft``).  No counterpart in the reference.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _C

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def verify_draft(target_probs: torch.Tensor, draft_probs: Optional[torch.Tensor], draft_tokens: torch.Tensor,
                 accept_u: torch.Tensor, sample_u: torch.Tensor, n_draft: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None):
    """Accept drafted tokens against the target's probabilities and draw the token after them.

    target_probs  (B, K+1, V) fp32, fp16 or bf16: row j is the target's distribution after j drafts
    draft_probs   (B, K, V) of the same type, or None for drafts without a distribution (q = 1)
    draft_tokens  (B, K) int64;  n_draft (B,) int32: drafts of each sequence (None: K)
    accept_u      (B, K) and sample_u (B,) fp32: uniform numbers in [0, 1)

    Draft j is kept while accept_u * q(x) < p(x).  The next token is drawn by sample_u from max(p - q, 0) at
    the first rejected draft, or from p after the last: the accepted tokens and it are distributed as the
    target's own samples.  Probabilities are counted in whole units of 2^-40, so the result depends on the
    inputs alone.  Returns (accepted int32 (B,), tokens int64 (B, K+1): kept drafts, the next token, then -1).
    A drafted token outside the vocabulary counts as rejected and sets ``status`` (int32 (1,)) if given."""
    p, q, x = target_probs, draft_probs, draft_tokens
    dt = _DTYPES.get(p.dtype)
    if dt is None:
        raise TypeError(f"probabilities must be fp32, fp16 or bf16 (got {p.dtype})")
    dev = p.device
    if dev.type != "cuda":
        raise RuntimeError("akv: verify_draft runs on CUDA tensors only (no CPU fallback)")
    index = _C.current_device()
    if dev.index is not None and dev.index != index:  # launches go to the current GPU
        with torch.cuda.device(dev.index):
            return verify_draft(p, q, x, accept_u, sample_u, n_draft, status)
    if p.dim() != 3 or x.dim() != 2:
        raise ValueError("target_probs must be (B, K+1, V) and draft_tokens (B, K)")
    B, K1, V = p.shape
    K = K1 - 1
    if x.shape != (B, K) or x.dtype is not torch.int64 or x.device != dev:
        raise ValueError(f"draft_tokens must be int64 ({B}, {K}) on {dev}")
    ps, qp, qs = p.stride(), 0, (0, 0, 1)
    if ps[2] != 1:
        p = p.contiguous()
        ps = p.stride()
    if q is not None:
        if q.shape != (B, K, V) or q.dtype is not p.dtype or q.device != dev:
            raise ValueError(f"draft_probs must be ({B}, {K}, {V}) {p.dtype} on {dev}")
        qs = q.stride()
        if qs[2] != 1:
            q = q.contiguous()
            qs = q.stride()
        if K:
            qp = q.data_ptr()
    au, su = accept_u, sample_u
    if au.shape != (B, K) or su.shape != (B,) or au.dtype is not torch.float32 or su.dtype is not torch.float32 or \
            au.device != dev or su.device != dev:
        raise ValueError(f"accept_u ({B}, {K}) and sample_u ({B},) must be fp32 on {dev}")
    nd = n_draft
    if nd is not None:
        if nd.shape != (B,) or nd.dtype is not torch.int32 or nd.device != dev:
            raise ValueError(f"n_draft must be int32 ({B},) on {dev}")
        nd = nd.contiguous()
    if status is not None and (status.dtype is not torch.int32 or status.device != dev):
        raise ValueError(f"status must be int32 on {dev}")
    x, au, su = x.contiguous(), au.contiguous(), su.contiguous()
    # empty_strided: 1.5 us of host time, torch.empty with its keywords 2.3
    accepted = torch.empty_strided((B,), (1,), dtype=torch.int32, device=dev)
    out = torch.empty_strided((B, K1), (K1, 1), dtype=torch.int64, device=dev)
    rc = _C.load().akv_verify_draft(
        _C.VERIFY_ARGS.pack(p.data_ptr(), ps[0], ps[1], qp, qs[0], qs[1], x.data_ptr(),
                            0 if nd is None else nd.data_ptr(), au.data_ptr(), su.data_ptr(), accepted.data_ptr(),
                            out.data_ptr(), 0 if status is None else status.data_ptr(), B, K, V, dt),
        _C.raw_stream(index))
    if rc:
        _C.check(rc, "akv_verify_draft")
    return accepted, out
