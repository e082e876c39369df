"""Texts longer than the cache: chunks in, light tokens out, every token's log probability.

A small random-init decoder scores a batch of texts chunk by chunk over an
``Int4PagedCache`` whose rows never hold more than ``keep`` tokens between
chunks.  Of a chunk, ``attend_chunk`` computes the attention, ``weigh`` adds what
each cached token got of it, and ``evict`` drops the tokens that got least; the
first ones and the latest stay.  ``token_logprobs`` gives the log probability,
entropy and rank of each of the text's own tokens.  The texts are then continued
token by token in the same way.  Nothing waits for the host.

    python adaptive-kv-memory_b200/examples/bounded_context.py
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import akv  # noqa: E402
from speculative_decode import Decoder  # noqa: E402


class BoundedDecoder(Decoder):
    def cache(self, max_seqs: int, max_tokens: int, n_pages: int) -> "akv.Int4PagedCache":
        return akv.Int4PagedCache(len(self.layers), n_pages, self.kv_heads, self.head_dim, group_size=32,
                                  max_seqs=max_seqs, max_blocks=-(-max_tokens // 32), device=self.device,
                                  track_weights=True)

    def forward(self, tokens, cache, rows, first_pos, n_new=None):
        """Logits (R, M, vocab) fp32 of row i's next n_new[i] (None: M) tokens, at positions first_pos onwards: rows
        that lost tokens are shorter than their texts.  Past n_new[i] they mean nothing."""
        R, M = tokens.shape
        new = cache.reserve(rows, M if n_new is None else n_new)
        pos = (first_pos + torch.arange(M, device=tokens.device)).float()[None].expand(R, M)
        attend = cache.attend if M == 1 else cache.attend_chunk
        x = self.embed[tokens]
        for i, p in enumerate(self.layers):
            q, k, v = (self._norm(x) @ p["qkv"]).view(R, M, -1, self.head_dim).transpose(1, 2).split(
                [self.heads, self.kv_heads, self.kv_heads], 1)
            q = self._rope(q, pos)
            cache.append(i, self._rope(k, pos), v, rows, new)
            a, lse = attend(i, q, rows, new, return_lse=True)
            cache.weigh(i, q, lse, rows, new)
            x = x + a.transpose(1, 2).reshape(R, M, -1) @ p["o"]
            u = self._norm(x) @ p["up"]
            x = x + torch.nn.functional.silu(u) @ p["down"]
        return (self._norm(x) @ self.head).float()


def score(model, texts, lengths, chunk=256, keep=512, first=4, recent=128, more=16):
    """Log probabilities of the texts' tokens (R, L), of which row i has lengths[i], each given those before it; then
    ``more`` further tokens, the best one each time.  Returns (TokenLogprobs of tokens 1 .. L - 1, NaN past a text's
    end; the new tokens (R, more); the cache)."""
    R, L = texts.shape
    dev = texts.device
    rows = torch.arange(R, dtype=torch.int32, device=dev)
    cache = model.cache(R, keep + max(chunk, more), R * (-(-(keep + max(chunk, more)) // 32) + 1))
    parts, last = [], torch.zeros(R, model.vocab, device=dev)
    for at in range(0, L, chunk):
        ids = texts[:, at:at + chunk]
        M = ids.shape[1]
        n_new = (lengths - at).clamp(0, M).to(torch.int32)
        logits = model.forward(ids, cache, rows, at, n_new)
        # token t + 1's, -1 (no token: NaN) past the end
        following = torch.nn.functional.pad(texts[:, at + 1:at + 1 + M], (0, M), value=-1)[:, :M]
        there = at + 1 + torch.arange(M, device=dev)[None] < lengths[:, None]
        parts.append(akv.token_logprobs(logits, torch.where(there, following, -1)))
        ends = (n_new > 0) & (lengths <= at + M)
        final = logits[torch.arange(R, device=dev), (n_new - 1).clamp_min(0).long()]
        last = torch.where(ends[:, None], final, last)
        cache.evict(rows, keep, first=first, recent=recent)
    scored = akv.TokenLogprobs(*(torch.cat([getattr(p, f) for p in parts], 1)[:, :L - 1]
                                 for f in ("logprob", "entropy", "rank")), None, None)
    out = []
    for step in range(more):
        best = akv.token_logprobs(last, torch.zeros(R, dtype=torch.int64, device=dev), top=1).top_tokens
        out.append(best)
        # (texts of several lengths go on at the longest one's position: their keys keep their own)
        last = model.forward(best, cache, rows, L + step)[:, 0]
    cache.evict(rows, keep, first=first, recent=recent)
    cache.check()
    return scored, torch.cat(out, 1) if out else texts[:, :0], cache


def main() -> None:
    model = BoundedDecoder()
    g = torch.Generator("cuda").manual_seed(1)
    lengths = torch.tensor([2000, 1500, 700, 2000], device="cuda")
    texts = torch.randint(0, model.vocab, (4, 2000), device="cuda", generator=g)
    scored, new, cache = score(model, texts, lengths)
    mean = torch.nanmean(scored.logprob, 1)
    print("mean log probability a token", [round(x, 3) for x in mean.tolist()])
    print(f"tokens held a row {cache.lens.tolist()} of {[n + new.shape[1] for n in lengths.tolist()]}, "
          f"{int((cache.refs > 0).sum())} of {cache.n_pages} pages live")


if __name__ == "__main__":
    main()
