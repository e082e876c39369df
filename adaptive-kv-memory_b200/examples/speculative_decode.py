"""Speculative decoding over the 4-bit paged cache, several continuations a prompt.

A small random-init decoder (the target) and its first layers (the draft)
each keep an ``Int4PagedCache``.  Every prompt is run once; ``fork`` gives it
``n`` continuations that share its pages.  A step drafts ``k`` tokens with the
draft model, scores them and the token before them in one target pass,
``verify_draft`` keeps the accepted ones and draws the next, and ``truncate``
rolls both caches back to what was kept.  Page tables, lengths and accepted
counts stay on the device: no step waits for the host.

    python adaptive-kv-memory_b200/examples/speculative_decode.py
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import akv  # noqa: E402


class Decoder:
    """Pre-norm decoder layers with grouped-query attention over an ``Int4PagedCache``."""

    def __init__(self, layers=4, hidden=512, heads=8, kv_heads=2, head_dim=64, vocab=1000, seed=0,
                 dtype=torch.bfloat16, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def w(*shape):
            return (torch.randn(*shape, generator=g, device=device) / shape[0] ** 0.5).to(dtype)

        self.heads, self.kv_heads, self.head_dim, self.vocab, self.device = heads, kv_heads, head_dim, vocab, device
        self.embed = w(vocab, hidden) * vocab ** 0.5
        self.layers = [dict(qkv=w(hidden, (heads + 2 * kv_heads) * head_dim), o=w(heads * head_dim, hidden),
                            up=w(hidden, 2 * hidden), down=w(2 * hidden, hidden) * 0.5) for _ in range(layers)]
        self.head = w(hidden, vocab) * 4

    def first(self, n: int) -> "Decoder":
        """A draft model: the first n layers, the same embedding and head."""
        d = object.__new__(Decoder)
        d.__dict__.update(self.__dict__, layers=self.layers[:n])
        return d

    def cache(self, max_seqs: int, max_tokens: int, n_pages: int) -> "akv.Int4PagedCache":
        return akv.Int4PagedCache(len(self.layers), n_pages, self.kv_heads, self.head_dim, group_size=32,
                                  max_seqs=max_seqs, max_blocks=-(-max_tokens // 32), device=self.device)

    def _rope(self, x, pos):
        half = self.head_dim // 2
        ang = pos[:, None, :, None] * (10000.0 ** (-torch.arange(half, device=x.device) / half))
        a, b = x.float().chunk(2, -1)
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1).to(x.dtype)

    @staticmethod
    def _norm(x):
        f = x.float()
        return (f * (f.square().mean(-1, keepdim=True) + 1e-6).rsqrt()).to(x.dtype)

    def forward(self, tokens, cache, rows):
        """Logits (R, M, vocab) fp32 of M new tokens per row, their K / V appended to the cache."""
        R, M = tokens.shape
        new = cache.reserve(rows, M)
        pos = ((cache.lens[rows.long()] - new)[:, None] + torch.arange(M, device=tokens.device)).float()
        x = self.embed[tokens]
        for i, p in enumerate(self.layers):
            q, k, v = (self._norm(x) @ p["qkv"]).view(R, M, -1, self.head_dim).transpose(1, 2).split(
                [self.heads, self.kv_heads, self.kv_heads], 1)
            cache.append(i, self._rope(k, pos), v, rows, new)
            a = cache.attend(i, self._rope(q, pos), rows, new)
            x = x + a.transpose(1, 2).reshape(R, M, -1) @ p["o"]
            u = self._norm(x) @ p["up"]
            x = x + torch.nn.functional.silu(u) @ p["down"]
        return (self._norm(x) @ self.head).float()


def probabilities(logits, temperature):
    """Next-token probabilities; temperature 0 puts all of it on the best token."""
    if temperature == 0:
        return torch.zeros_like(logits).scatter_(-1, logits.argmax(-1, keepdim=True), 1.0)
    return torch.softmax(logits / temperature, -1)


def speculative_generate(target, draft, prompts, n=2, steps=8, k=4, temperature=0.8, seed=0):
    """Continue every prompt (P, L) n times.  Returns (tokens (P*n, L + generated), -1 padded; accepted counts
    (steps, P*n); the target's cache), all still on the device."""
    P, L = prompts.shape
    R, dev = P * n, prompts.device
    g = torch.Generator(device=dev).manual_seed(seed)
    room = L + steps * (k + 1) + 1
    pages = P * -(-L // 32) + R * (-(-room // 32) + 1)
    tc, dc = target.cache(R, room + k + 1, pages), draft.cache(R, room + k + 1, pages)
    first = torch.arange(0, R, n, dtype=torch.int32, device=dev)          # the rows that run the prompts
    rows = torch.arange(R, dtype=torch.int32, device=dev)
    kids = rows[rows % n != 0]
    # all but the prompt's last token go into the caches once; the continuations share their pages
    for model, cache in ((target, tc), (draft, dc)):
        model.forward(prompts[:, :-1], cache, first)
        if n > 1:
            cache.fork(kids - kids % n, kids)
    last = prompts[:, -1:].repeat_interleave(n, 0)
    out, counts = [prompts.repeat_interleave(n, 0)], []
    for _ in range(steps):
        base = tc.lens.clone()
        toks, probs = [last], []
        for _ in range(k):
            q = probabilities(draft.forward(toks[-1], dc, rows)[:, -1], temperature)
            noise = -torch.rand(q.shape, generator=g, device=dev).clamp_min(1e-30).log()
            toks.append((q / noise).argmax(-1, keepdim=True))
            probs.append(q)
        draft.forward(toks[-1], dc, rows)                                 # the last draft's K / V
        p = probabilities(target.forward(torch.cat(toks, 1), tc, rows), temperature)
        accepted, kept = akv.verify_draft(p, torch.stack(probs, 1), torch.cat(toks[1:], 1),
                                          torch.rand(R, k, generator=g, device=dev),
                                          torch.rand(R, generator=g, device=dev))
        keep = base + accepted + 1
        tc.truncate(rows, keep)
        dc.truncate(rows, keep)
        last = kept.gather(1, accepted.long()[:, None])
        out.append(kept)
        counts.append(accepted)
    tc.check()
    dc.check()
    return torch.cat(out, 1), torch.stack(counts), tc


def main() -> None:
    target = Decoder()
    draft = target.first(2)
    prompts = torch.randint(0, target.vocab, (4, 45), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    tokens, accepted, cache = speculative_generate(target, draft, prompts, n=4, steps=12)
    print(f"{tokens.shape[0]} continuations, {accepted.float().mean().item():.2f} of 4 drafted tokens kept a step, "
          f"{int((tokens >= 0).sum()) - prompts.numel() * 4} tokens")
    cache.free(torch.arange(1, tokens.shape[0], 2, dtype=torch.int32, device="cuda"))
    live = int(cache.compact())
    cache.check()
    print(f"half of them freed: {live} of {cache.n_pages} pages live, packed at the pool's low end")


if __name__ == "__main__":
    main()
