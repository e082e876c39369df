"""Log probabilities of given tokens, with entropy, rank and the top alternatives.

``token_logprobs`` reads every row of logits once (``akv_token_logprobs``): a
prompt's tokens scored after a chunk, or a step's sampled tokens with their
alternatives.  No counterpart in the reference.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _C

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor        # fp32, the tokens' shape
    entropy: torch.Tensor        # fp32, the tokens' shape
    rank: torch.Tensor           # int32, the tokens' shape
    top_tokens: torch.Tensor     # int64, the tokens' shape and (top,)
    top_logprobs: torch.Tensor   # fp32, alike


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """What the softmax of each row of logits says of its token.

    logits (..., V) fp32, fp16 or bf16;  tokens (...) int64;  top 0 to 32 alternatives (at most V)

    ``logprob`` of the token, ``entropy`` of the row (nats), ``rank`` of the token (1 + the logits above its own),
    and the ``top`` largest logits' tokens in descending order (the lowest token first among equal ones) with their
    log probabilities.  A logit of -inf has probability 0.  A token outside [0, V) gives logprob NaN and rank 0; a
    row without a distribution (NaN or +inf in it, or -inf alone) NaN everywhere, rank 0 and top tokens -1."""
    dt = _DTYPES.get(logits.dtype)
    if dt is None:
        raise TypeError(f"logits must be fp32, fp16 or bf16 (got {logits.dtype})")
    dev = logits.device
    if dev.type != "cuda":
        raise RuntimeError("akv: token_logprobs runs on CUDA tensors only (no CPU fallback)")
    index = _C.current_device()
    if dev.index is not None and dev.index != index:  # launches go to the current GPU
        with torch.cuda.device(dev.index):
            return token_logprobs(logits, tokens, top)
    shape = logits.shape
    if not shape or tokens.shape != shape[:-1] or tokens.dtype is not torch.int64 or tokens.device != dev:
        raise ValueError(f"logits must be (..., V) and tokens int64 {tuple(shape[:-1])} on {dev}")
    V = shape[-1]
    if not 0 <= top <= min(MAX_TOP, V) or V == 0:
        raise ValueError(f"top must be 0 to {min(MAX_TOP, V)} (got {top}), and V positive")
    x = logits if len(shape) == 2 else logits.reshape(-1, V)
    stride, inner = x.stride()
    if inner != 1 and V > 1:
        x = x.contiguous()
        stride = V
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    n, lead = x.shape[0], tokens.shape
    # empty_strided: 1.5 us of host time, torch.empty with its keywords 2.3
    row = tokens.stride()
    logprob = torch.empty_strided(lead, row, dtype=torch.float32, device=dev)
    entropy = torch.empty_strided(lead, row, dtype=torch.float32, device=dev)
    rank = torch.empty_strided(lead, row, dtype=torch.int32, device=dev)
    many = tuple(s * top for s in row) + (1,)
    ids = torch.empty_strided((*lead, top), many, dtype=torch.int64, device=dev)
    alt = torch.empty_strided((*lead, top), many, dtype=torch.float32, device=dev)
    rc = _C.load().akv_token_logprobs(
        _C.LOGPROBS_ARGS.pack(x.data_ptr(), stride, tokens.data_ptr(), logprob.data_ptr(), entropy.data_ptr(),
                              rank.data_ptr(), ids.data_ptr(), alt.data_ptr(), n, V, top, dt), _C.raw_stream(index))
    if rc:
        _C.check(rc, "akv_token_logprobs")
    return TokenLogprobs(logprob, entropy, rank, ids, alt)
