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
    _C.require_cuda(target_probs, draft_probs, draft_tokens, accept_u, sample_u, n_draft)
    if target_probs.dtype not in _DTYPES:
        raise TypeError(f"probabilities must be fp32, fp16 or bf16 (got {target_probs.dtype})")
    if target_probs.dim() != 3 or draft_tokens.dim() != 2:
        raise ValueError("target_probs must be (B, K+1, V) and draft_tokens (B, K)")
    B, K1, V = target_probs.shape
    K = K1 - 1
    if tuple(draft_tokens.shape) != (B, K) or draft_tokens.dtype != torch.int64:
        raise ValueError(f"draft_tokens must be int64 ({B}, {K})")
    if draft_probs is not None and (tuple(draft_probs.shape) != (B, K, V) or draft_probs.dtype != target_probs.dtype):
        raise ValueError(f"draft_probs must be ({B}, {K}, {V}) {target_probs.dtype}")
    if tuple(accept_u.shape) != (B, K) or tuple(sample_u.shape) != (B,) or accept_u.dtype != torch.float32 or \
            sample_u.dtype != torch.float32:
        raise ValueError(f"accept_u ({B}, {K}) and sample_u ({B},) must be fp32")
    if n_draft is not None and (tuple(n_draft.shape) != (B,) or n_draft.dtype != torch.int32):
        raise ValueError(f"n_draft must be int32 ({B},)")
    for t in (draft_probs, draft_tokens, accept_u, sample_u, n_draft, status):
        if t is not None and t.device != target_probs.device:
            raise ValueError("all tensors must be on one device")
    p = target_probs if target_probs.stride(-1) == 1 else target_probs.contiguous()
    q = draft_probs
    if q is not None and q.stride(-1) != 1:
        q = q.contiguous()
    tokens, au, su = draft_tokens.contiguous(), accept_u.contiguous(), sample_u.contiguous()
    nd = None if n_draft is None else n_draft.contiguous()
    accepted = torch.empty(B, dtype=torch.int32, device=p.device)
    out = torch.empty(B, K1, dtype=torch.int64, device=p.device)
    has_q = q is not None and K > 0
    rc = _C.load().akv_verify_draft(p.data_ptr(), p.stride(0), p.stride(1),
                                    q.data_ptr() if has_q else None, q.stride(0) if has_q else 0,
                                    q.stride(1) if has_q else 0, tokens.data_ptr(), _C.ptr(nd), au.data_ptr(),
                                    su.data_ptr(), B, K, V, _DTYPES[p.dtype], accepted.data_ptr(), out.data_ptr(),
                                    _C.ptr(status), _C.stream_of(p))
    _C.check(rc, "akv_verify_draft")
    return accepted, out
