"""Measured cases of long prompts and long conversations over the 4-bit paged cache in bounded memory.

Four operators, each reached as a serving program reaches it:

* ``chunk``   attention of a prompt's chunk (tens to thousands of new tokens a sequence) over the paged cache
* ``weigh``   the attention weight that each cached token receives from the new tokens, added to its running total
* ``evict``   the lightest tokens of each sequence dropped and the others moved together, in all layers
* ``logp``    log probabilities of given tokens, with entropy, rank and the top alternatives

``own`` False runs their plain form (elementary torch operations in 32 bits), True the framework's kernels.

The cache: page p of layer l holds, for each KV head, a record of 32 tokens: K codes [32][D/2] bytes (channel 2j in the
high nibble of byte j), V codes [32][D/2], then (scale, zero) fp16 pairs of K [32][G][2] and of V [32][G][2], with
G = D / group.  A code c of a group stands for c * scale + zero.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 32
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a short message continuing one conversation of 1K tokens, 12 query / 2 KV heads: latency
        dict(name="chunk_message_1k", op="chunk", rows=1, hq=12, hkv=2, dim=128, group=128, m=64, lo=1100, hi=1100,
             dtype="bfloat16"),
        # first chunks of four prompts of odd lengths (nothing cached before them), 32 / 8 heads, groups of 64
        dict(name="chunk_prompts_2k", op="chunk", rows=4, hq=32, hkv=8, dim=128, group=64, m=2047, lo=0, hi=0,
             dtype="float16"),
        # continuous batching: 16 sequences of 0.5K to 6K tokens with up to 256 new ones each, heads of 64
        dict(name="chunk_ragged_16", op="chunk", rows=16, hq=24, hkv=8, dim=64, group=16, m=256, lo=500, hi=6000,
             dtype="bfloat16"),
        # the sixteenth 2K chunk of two prompts of 32K tokens
        dict(name="chunk_long_32k", op="chunk", rows=2, hq=32, hkv=8, dim=128, group=128, m=2048, lo=32768, hi=32768,
             dtype="bfloat16"),
        # one conversation, one new token: the step of a small model's layer
        dict(name="weigh_one_4k", op="weigh", rows=1, hq=12, hkv=2, dim=128, group=128, m=1, lo=4096, hi=4096,
             dtype="float16"),
        # a full batch of long contexts, one token each
        dict(name="weigh_batch_32k", op="weigh", rows=16, hq=32, hkv=8, dim=128, group=128, m=1, lo=32768, hi=32768,
             dtype="float16"),
        # a prompt's chunk of 1,000 tokens over 16K
        dict(name="weigh_chunk_16k", op="weigh", rows=1, hq=32, hkv=8, dim=128, group=32, m=1000, lo=16001, hi=16001,
             dtype="bfloat16"),
        # one conversation of a small model (28 layers, 2 KV heads) brought back from 4,352 to 4,096 tokens
        dict(name="evict_one_4k", op="evict", kind="trim", layers=28, rows=1, hkv=2, dim=128, group=128, lo=4352,
             hi=4352, keep=4096, first=4, recent=256),
        # 16 sequences of 1K to 7K tokens in 16 layers of 8 heads, each brought down to 2,000
        dict(name="evict_batch_16", op="evict", kind="trim", layers=16, rows=16, hkv=8, dim=128, group=64, lo=1000,
             hi=7000, keep=2000, first=4, recent=128),
        # one sequence, one step: the sampled token's log probability and five alternatives
        dict(name="logp_step_1", op="logp", rows=1, vocab=151936, top=5, dtype="float32"),
        # a batch's step with 20 alternatives, odd vocabulary
        dict(name="logp_step_64", op="logp", rows=64, vocab=32003, top=20, dtype="bfloat16"),
        # a prompt scored: every token's log probability, entropy and best alternative
        dict(name="logp_prompt_4k", op="logp", rows=4093, vocab=151936, top=1, dtype="bfloat16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "weigh", "weigh", "evict", "logp"])
    if op == "logp":
        rows = _spread(rng, 1, 4096)
        return dict(op=op, rows=rows, vocab=_spread(rng, 1000, min(152000, 4093 * 151936 // rows)),
                    top=rng.choice([0, 1, 5, 20, rng.randint(2, 32)]),
                    dtype=rng.choice(["float32", "float16", "bfloat16"] if rows < 1024 else ["float16", "bfloat16"]))
    dim = rng.choice([64, 128, 128, 256])
    group = rng.choice([g for g in (16, 32, 64, 128, 256) if dim // 4 <= g <= dim])
    hkv = _spread(rng, 1, 8)
    if op == "evict":
        rows, layers = _spread(rng, 1, 32), _spread(rng, 1, 28)
        most = min(8192, 16 * 7000 * 16 * 8 * 128 // (rows * layers * hkv * dim) // 2)
        hi = _spread(rng, 64, max(64, most))
        first, recent = rng.choice([0, 1, 4]), _spread(rng, 1, max(1, hi // 8))
        return dict(op=op, kind=rng.choice(["trim", "trim", "fork"]), layers=layers, rows=rows, hkv=hkv, dim=dim,
                    group=group, lo=rng.choice([hi, hi // 4 + 1]), hi=hi, keep=_spread(rng, first + recent, hi),
                    first=first, recent=recent)
    hq = hkv * _spread(rng, 1, 8)
    rows = _spread(rng, 1, 16)
    m = _spread(rng, 16, 2048) if op == "chunk" else rng.choice([1, _spread(rng, 1, 1000)])
    # no more products, no more pairs of queries and tokens and no more cache than the largest listed case
    pairs = 2 * 32 * 2048 * 32768 if op == "chunk" else 32 * 1000 * 16001
    m = max(1, min(m, int(math.sqrt(pairs * 128 / (rows * hq * max(dim, 128)))) - 16))
    most = min(32768, pairs * 128 // (rows * hq * m * max(dim, 128)), 16 * 32768 * 8 * 128 // (rows * hkv * dim))
    hi = _spread(rng, 16, max(16, most - m))
    return dict(op=op, rows=rows, hq=hq, hkv=hkv, dim=dim, group=group, m=m, lo=rng.choice([0, hi, hi // 3]), hi=hi,
                dtype=rng.choice(["float16", "bfloat16"]))


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    return g


def _host(seed):
    g = torch.Generator()
    g.manual_seed((int(seed) * 7919 + 17) & 0x7FFFFFFFFFFF)
    return g


def _ints(lo, hi, n, g):
    return torch.randint(lo, hi + 1, (n,), generator=g, dtype=torch.int64)


def _record_bytes(dim, group):
    return BLOCK * (dim + 8 * (dim // group))


def _pack_rows(x, group):
    """Codes in bytes (…, D/2) and (scale, zero) pairs (…, G, 2) of rows x (…, D)."""
    g = x.unflatten(-1, (-1, group))
    lo = g.amin(-1).half()
    s = ((g.amax(-1) - lo.float()) / 15.0).half()
    c = ((g - lo.float().unsqueeze(-1)) / s.float().unsqueeze(-1)).round().clamp(0, 15).flatten(-2).to(torch.uint8)
    return (c[..., 0::2] << 4) | c[..., 1::2], torch.stack([s, lo], -1)


def _direction(dim, seed):
    """What a model's queries have in common: tokens whose keys point there are looked at by all of them."""
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) % 1000003 + 5)
    return torch.sign(torch.randn(dim, generator=g, device=DEV)) * 0.5


def _fields(buf, dim, group):
    """Views of a (…, rec) uint8 buffer: K codes, V codes (…, 32, D/2), K and V (scale, zero) (…, 32, G, 2) fp16."""
    h, n = BLOCK * dim // 2, BLOCK * (dim // group) * 4
    kc = buf[..., :h].unflatten(-1, (BLOCK, dim // 2))
    vc = buf[..., h:2 * h].unflatten(-1, (BLOCK, dim // 2))
    kp = buf[..., 2 * h:2 * h + n].view(torch.float16).unflatten(-1, (BLOCK, dim // group, 2))
    vp = buf[..., 2 * h + n:].view(torch.float16).unflatten(-1, (BLOCK, dim // group, 2))
    return kc, vc, kp, vp


def _tables(lens, n_pages, max_blocks, g):
    """A page table for these lengths over shuffled pages (-1 where a row has none)."""
    perm = torch.randperm(n_pages, generator=g)
    table = torch.full((len(lens), max_blocks), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(lens):
        nb = -(-n // BLOCK)
        table[r, :nb] = perm[at:at + nb].int()
        at += nb
    return table


def _attention_inputs(case, seed):
    """Quantised pages of every row, queries as a projection gives them, the running weights."""
    g, hg = _gen(seed), _host(seed)
    dt = getattr(torch, case["dtype"])
    rows, m, hq, hkv, dim, group = (case[k] for k in ("rows", "m", "hq", "hkv", "dim", "group"))
    # lengths before the new tokens, and how many of them each row has
    before = _ints(case["lo"], case["hi"], rows, hg).tolist()
    ragged = rows > 1 and (case["lo"] < case["hi"] or case["hi"] == 0)
    new = _ints(max(1, m // 2), m, rows, hg).tolist() if ragged else [m] * rows
    if ragged:
        new[0] = m
    if case["lo"] == case["hi"] and case["hi"]:
        before = [n - m if n > m else n for n in before]  # the named length counts the new tokens
    lens = [a + b for a, b in zip(before, new)]
    max_blocks = -(-(case["hi"] + m) // BLOCK)
    n_pages = sum(-(-n // BLOCK) for n in lens) + 3
    table = _tables(lens, n_pages, max_blocks, hg)
    buf = torch.zeros(1, n_pages, hkv, _record_bytes(dim, group), dtype=torch.uint8, device=DEV)
    u = _direction(dim, seed)
    for r, n in enumerate(lens):
        nb = -(-n // BLOCK)
        rec = torch.empty(nb, hkv, buf.shape[3], dtype=torch.uint8, device=DEV)
        kc, vc, kp, vp = _fields(rec, dim, group)
        k = torch.randn(nb, hkv, BLOCK, dim, generator=g, device=DEV)
        k[..., 3] *= 6                      # a few channels of K are several times larger
        k[..., dim // 2 + 1] *= 4
        # some tokens draw every query's attention
        k += torch.randn(nb, 1, BLOCK, 1, generator=g, device=DEV).abs() * u
        for x, c, p in ((k, kc, kp), (torch.randn(nb, hkv, BLOCK, dim, generator=g, device=DEV), vc, vp)):
            code, pair = _pack_rows(x, group)
            c.copy_(code)
            p.copy_(pair)
        buf[0, table[r, :nb].to(DEV).long()] = rec
    q = (torch.randn(rows, m, hq, dim, generator=g, device=DEV) + 0.6 * u).to(dt).transpose(1, 2)
    d = dict(op=case["op"], buf=buf, table=table.to(DEV), lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
             new=torch.tensor(new, dtype=torch.int32, device=DEV), dim=dim, group=group, dtype=dt, hkv=hkv, q=q)
    if case["op"] == "weigh":
        # attention's log-sum-exp, as it returned it, and what the tokens have received before
        d["lse"] = _lse(d)
        d["weights"] = torch.rand(1, rows, max_blocks * BLOCK, generator=g, device=DEV).pow_(8)
    return d


def _evict_inputs(case, seed):
    g, hg = _gen(seed), _host(seed)
    rows, layers, dim, group = case["rows"], case["layers"], case["dim"], case["group"]
    lens = _ints(case["lo"], case["hi"], rows, hg).tolist()
    lens[0] = case["hi"]
    fork = case["kind"] == "fork"
    max_seqs = rows * (2 if fork else 1)
    max_blocks = -(-case["hi"] // BLOCK) + 1
    n_pages = rows * -(-case["hi"] // BLOCK) + 3 + (rows * (-(-case["keep"] // BLOCK) + 1) if fork else 0)
    table = torch.full((max_seqs, max_blocks), -1, dtype=torch.int32)
    table[:rows] = _tables(lens, n_pages, max_blocks, hg)
    all_lens = torch.zeros(max_seqs, dtype=torch.int32)
    all_lens[:rows] = torch.tensor(lens, dtype=torch.int32)
    buf = torch.randint(0, 256, (layers, n_pages, case["hkv"], _record_bytes(dim, group)), generator=g, device=DEV,
                        dtype=torch.uint8)
    # a token's total is heavy-tailed: most of the weight lies on few of them, the same ones in many layers
    w = (torch.randn(1, max_seqs, max_blocks * BLOCK, generator=g, device=DEV) * 2.0).exp()
    w = w * torch.rand(layers, max_seqs, max_blocks * BLOCK, generator=g, device=DEV)
    return dict(op="evict", kind=case["kind"], buf=buf, table=table.to(DEV), lens=all_lens.to(DEV), dim=dim,
                group=group, hkv=case["hkv"], rows=rows, keep=case["keep"], first=case["first"],
                recent=case["recent"], weights=w, parents=torch.arange(rows, dtype=torch.int32, device=DEV),
                kids=torch.arange(rows, 2 * rows, dtype=torch.int32, device=DEV))


def _logp_inputs(case, seed):
    g = _gen(seed)
    n, vocab = case["rows"], case["vocab"]
    dt = getattr(torch, case["dtype"])
    logits = torch.empty(n, vocab, dtype=dt, device=DEV)
    step = max(1, (1 << 26) // vocab)
    tokens = torch.empty(n, dtype=torch.int64, device=DEV)
    for a in range(0, n, step):
        b = min(n, a + step)
        # a model's logits: some rows nearly certain, others flat; the token mostly a likely one
        x = torch.randn(b - a, vocab, generator=g, device=DEV)
        x *= 1.0 + 3.0 * torch.rand(b - a, 1, generator=g, device=DEV)
        logits[a:b] = x.to(dt)
        near = x[:, :4096].argmax(-1)
        some = torch.randint(0, vocab, (b - a,), generator=g, device=DEV)
        tokens[a:b] = torch.where(torch.rand(b - a, generator=g, device=DEV) < 0.8, near, some)
    return dict(op="logp", logits=logits, tokens=tokens, top=case["top"])


def _inputs(case, seed):
    """The case's data, from the seed alone (plain tensors; no handle of the framework)."""
    return {"chunk": _attention_inputs, "weigh": _attention_inputs, "evict": _evict_inputs,
            "logp": _logp_inputs}[case["op"]](case, seed)


def prepare(case, seed):
    d = _inputs(case, seed)
    d["own"] = own
    if d["op"] == "evict":
        d.update(refs=_count_refs(d["table"], d["buf"].shape[1]), w0=d["weights"].clone())
        d.update(table0=d["table"].clone(), lens0=d["lens"].clone(), refs0=d["refs"].clone())
    if not own or d["op"] == "logp":
        return d
    table = d["table"]
    cache = _akv().Int4PagedCache(d["buf"].shape[0], d["buf"].shape[1], d["hkv"], d["dim"], group_size=d["group"],
                                  max_seqs=table.shape[0], max_blocks=table.shape[1], device=DEV,
                                  track_weights=d["op"] != "chunk")
    cache.load_state(d.pop("buf"), table, d["lens"])
    if d["op"] != "chunk":
        cache.weights.copy_(d.pop("weights"))
    if d["op"] == "evict":
        d["state0"] = cache.page_state()
    d["cache"] = cache
    return d


def _akv():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "adaptive-kv-memory_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import akv
    return akv


def _count_refs(table, n_pages):
    t = table.flatten().long()
    return torch.zeros(n_pages + 1, dtype=torch.int32, device=t.device).index_add_(
        0, torch.where(t < 0, n_pages, t), torch.ones_like(t, dtype=torch.int32))[:n_pages]


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if state["own"]:
        return _run_own(state)
    return {"chunk": _plain_chunk, "weigh": _plain_weigh, "evict": _plain_evict, "logp": _plain_logp}[state["op"]](state)


def _run_own(s):
    op = s["op"]
    if op == "logp":
        r = _akv().token_logprobs(s["logits"], s["tokens"], top=s["top"])
        return dict(logprob=r.logprob, entropy=r.entropy, rank=r.rank, top_tokens=r.top_tokens,
                    top_logprobs=r.top_logprobs)
    c = s["cache"]
    if op == "chunk":
        return dict(out=c.attend_chunk(0, s["q"], n_new=s["new"]))
    if op == "weigh":
        c.weigh(0, s["q"], s["lse"], n_new=s["new"])
        return dict(weights=c.weights)
    c.weights.copy_(s["w0"])
    if s["kind"] == "fork":
        # a trimmed copy of every sequence; the sequences themselves stay as they are
        c.fork(s["parents"], s["kids"])
        kept = c.evict(s["kids"], s["keep"], first=s["first"], recent=s["recent"])
        table, lens, refs = c.table.clone(), c.lens.clone(), c.refs.clone()
        c.free(s["kids"])
        return dict(kept=kept, table=table, lens=lens, refs=refs, weights=c.weights, buf=c.buf)
    c.set_page_state(s["state0"])
    kept = c.evict(s["parents"], s["keep"], first=s["first"], recent=s["recent"])
    return dict(kept=kept, table=c.table, lens=c.lens, refs=c.refs, weights=c.weights, buf=c.buf)


# ------------------------------------------------------------------------------------------------ plain forms
def _values(codes, pairs, group):
    """fp32 values (…, D) of codes (…, D/2) bytes and (scale, zero) pairs (…, G, 2)."""
    c = torch.stack([codes >> 4, codes & 15], -1).flatten(-2).float().unflatten(-1, (-1, group))
    return (c * pairs[..., 0:1].float() + pairs[..., 1:2].float()).flatten(-2)


def _pages_of(s):
    """Codes and pairs of every row's tokens, (rows, hkv, blocks, 32, …)."""
    return _fields(s["buf"][0, s["table"].clamp_min(0).long()].transpose(1, 2), s["dim"], s["group"])


def _scores(s, kc, kp):
    """Scaled scores (rows, hkv, rep, m, tokens), -inf where a query does not see a token."""
    rows, hq, m, dim = s["q"].shape
    hkv = s["hkv"]
    q = s["q"].float().unflatten(1, (hkv, hq // hkv)).flatten(2, 3)
    x = (q @ _values(kc, kp, s["group"]).flatten(2, 3).transpose(2, 3)).unflatten(2, (hq // hkv, m))
    x /= math.sqrt(dim)
    i, t = torch.arange(m, device=q.device), torch.arange(x.shape[-1], device=q.device)
    new, n = s["new"].long(), s["lens"].long()
    seen = (t <= (n - new)[:, None, None] + i[None, :, None]) & (i[None, :] < new[:, None])[:, :, None]
    return x.masked_fill_(~seen[:, None, None], -math.inf)


def _plain_chunk(s):
    kc, vc, kp, vp = _pages_of(s)
    x = _scores(s, kc, kp)
    top = x.amax(-1, keepdim=True).clamp_min(-3.0e38)
    x.sub_(top).exp_()
    z = x.sum(-1, keepdim=True)
    out = x.flatten(2, 3) @ _values(vc, vp, s["group"]).flatten(2, 3)
    out = out.unflatten(2, x.shape[2:4]) / torch.where(z > 0, z, 1.0)
    return dict(out=out.flatten(1, 2).to(s["dtype"]))


def _lse(s):
    """Log-sum-exp (rows, hq, m) of attention over the cache; -inf past a row's new tokens."""
    outs = []
    for r in range(s["q"].shape[0]):
        one = dict(s, **{k: s[k][r:r + 1] for k in ("q", "table", "new", "lens")})
        kc, _, kp, _ = _pages_of(one)
        outs.append(torch.logsumexp(_scores(one, kc, kp), -1).flatten(1, 2))
    return torch.cat(outs)


def _plain_weigh(s):
    kc, _, kp, _ = _pages_of(s)
    x = _scores(s, kc, kp)
    lse = s["lse"].unflatten(1, x.shape[1:3]).unsqueeze(-1)
    x.sub_(torch.where(lse == -math.inf, 0.0, lse)).exp_()
    # rows that see nothing have scores of -inf alone: weight 0
    s["weights"][0] += x.sum((1, 2, 3))
    return dict(weights=s["weights"])


def _plain_evict(s):
    # the state a program evicts from: fresh page tables, the weights as they stand
    s["weights"].copy_(s["w0"])
    table, lens, refs, buf, w = s["table"], s["lens"], s["refs"], s["buf"], s["weights"]
    table.copy_(s["table0"])
    lens.copy_(s["lens0"])
    refs.copy_(s["refs0"])
    rows = s["parents"].long()
    if s["kind"] == "fork":
        kids = s["kids"].long()
        table[kids], lens[kids] = table[rows], lens[rows]
        w[:, kids] = torch.where(torch.arange(w.shape[2], device=w.device) < lens[rows][:, None], w[:, rows], w[:, kids])
        refs.copy_(_count_refs(table, refs.numel()))
        rows = kids
    n, keep = lens[rows].long(), s["keep"]
    t = torch.arange(w.shape[2], device=w.device)
    score = w[:, rows].double().sum(0).float()
    score = torch.where((t < s["first"]) | (t >= n[:, None] - s["recent"]), math.inf, score)
    score = torch.where(t < n[:, None], score, -math.inf)
    order = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :keep]
    left = n.clamp_max(keep)
    on = torch.arange(keep, device=w.device) < left[:, None]
    kept = torch.where(on, order, 1 << 40).sort(1).values
    # pages written: from the first token that moves; a shared one is left and a free one taken for it
    j = torch.arange(keep, device=w.device)
    src = torch.where(on, kept, j)
    blocks = torch.arange(table.shape[1], device=w.device)
    moves = on & (src != j)
    start = torch.where(moves.any(1), moves.int().argmax(1), 1 << 40)
    old = table[rows].long()
    written = (blocks >= (start // BLOCK)[:, None]) & (blocks < ((left + BLOCK - 1) // BLOCK)[:, None])
    shared = written & (refs[old.clamp_min(0)] > 1)
    free = (refs == 0).nonzero().flatten()
    new = old.clone()
    new[shared] = free[:int(shared.sum())]
    page = lambda tab, x: tab.gather(1, (x // BLOCK).clamp_max(tab.shape[1] - 1))  # noqa: E731
    live = on & (j >= (start // BLOCK * BLOCK)[:, None])
    r, c = live.nonzero(as_tuple=True)
    p0, s0, p1, s1 = page(old, src)[r, c], src[r, c] % BLOCK, page(new, j.expand_as(src))[r, c], j[c] % BLOCK
    for f in _fields(buf, s["dim"], s["group"]):
        f[:, p1, :, s1] = f[:, p0, :, s0]
    w[:, rows[r], j[c]] = w[:, rows[r], src[r, c]]
    gone = blocks >= ((left + BLOCK - 1) // BLOCK)[:, None]
    table[rows] = torch.where(gone, -1, new).int()
    lens[rows] = left.int()
    refs.copy_(_count_refs(table, refs.numel()))
    return dict(kept=torch.where(on, kept, -1).int(), table=table, lens=lens, refs=refs, weights=w, buf=buf)


def _ordered(x):
    """Whole numbers in the order of fp32 values x."""
    b = (x + 0.0).view(torch.int32)
    return b ^ ((b >> 31) & 0x7FFFFFFF)


def _plain_logp(s):
    x, k = s["logits"].float(), s["top"]
    n, vocab = x.shape
    top = x.amax(1, keepdim=True)
    mine = x.gather(1, s["tokens"][:, None])
    rank = (x > mine).sum(1) + 1
    if k:
        # the largest values, the lowest index first among equal ones
        key = (_ordered(x).long() << 32) | (vocab - 1 - torch.arange(vocab, device=x.device))
        ids = vocab - 1 - (key.topk(k, dim=1).values & 0xFFFFFFFF)
        del key
        best = x.gather(1, ids) - top
    x = x.sub_(top)
    e = x.exp()
    z = e.sum(1, keepdim=True)
    logz = z.log()
    entropy = logz - e.mul_(x).sum(1, keepdim=True) / z
    r = dict(logprob=(mine - top - logz).squeeze(1), entropy=entropy.squeeze(1), rank=rank.int())
    r["top_tokens"] = ids if k else torch.empty(n, 0, dtype=torch.int64, device=x.device)
    r["top_logprobs"] = best - logz if k else torch.empty(n, 0, device=x.device)
    return r


# ------------------------------------------------------------------------------------------------ 64 bits
def _row64(d, r):
    """K and V of row r in 64 bits, (hkv, len, D), from the bytes one field at a time."""
    dim, group, n = d["dim"], d["group"], int(d["lens"][r])
    rec = d["buf"][0, d["table"][r, :-(-n // BLOCK)].long()]
    out = []
    half, pairs = BLOCK * dim // 2, BLOCK * (dim // group) * 4
    for c0, p0 in ((0, 2 * half), (half, 2 * half + pairs)):
        code = rec[..., c0:c0 + half].reshape(*rec.shape[:2], BLOCK, dim // 2).to(torch.int32)
        x = torch.empty(*rec.shape[:2], BLOCK, dim, dtype=torch.float64, device=DEV)
        x[..., 0::2], x[..., 1::2] = (code // 16).double(), (code % 16).double()
        sz = rec[..., p0:p0 + pairs].contiguous().view(torch.float16).double().view(*rec.shape[:2], BLOCK, -1, 2)
        x = x * sz[..., 0].repeat_interleave(group, -1) + sz[..., 1].repeat_interleave(group, -1)
        out.append(x.transpose(0, 1).reshape(rec.shape[1], -1, dim)[:, :n])
    return out


def _exact_attention(d):
    rows, hq, m, dim = d["q"].shape
    rep = hq // d["hkv"]
    out = torch.zeros(rows, hq, m, dim, dtype=torch.float64, device=DEV)
    w = d["weights"].double() if d["op"] == "weigh" else None
    for r in range(rows):
        n, new = int(d["lens"][r]), int(d["new"][r])
        k, v = _row64(d, r)
        mask = torch.arange(n, device=DEV)[None] > (n - new + torch.arange(new, device=DEV))[:, None]
        for h in range(hq):
            x = d["q"][r, h, :new].double() @ k[h // rep].T * dim ** -0.5
            x.masked_fill_(mask, -math.inf)
            if w is None:
                out[r, h, :new] = torch.softmax(x, -1) @ v[h // rep]
            else:
                w[0, r, :n] += torch.exp(x - d["lse"][r, h, :new, None].double()).sum(0)
    return dict(out=out) if w is None else dict(weights=w)


def _exact_evict(d):
    """The weights as they stand after the eviction; everything else is whole numbers."""
    w, lens = d["weights"].cpu().numpy().astype(np.float64), d["lens"].cpu().numpy()
    for r in range(d["rows"]):
        n, to = int(lens[r]), r
        if d["kind"] == "fork":
            to = d["rows"] + r
            w[:, to, :n] = w[:, r, :n]
        if n <= d["keep"]:
            continue
        score = w[:, to, :n].sum(0).astype(np.float32)
        forced = [t for t in range(n) if t < d["first"] or t >= n - d["recent"]]
        rest = sorted((t for t in range(n) if d["first"] <= t < n - d["recent"]), key=lambda t: (-score[t], t))
        kept = sorted(forced + rest[:d["keep"] - len(forced)])
        w[:, to, :d["keep"]] = w[:, to][:, kept]
    return dict(kept=None, table=None, lens=None, refs=None, weights=torch.from_numpy(w), buf=None)


def _exact_logp(d):
    n, k = d["logits"].shape[0], d["top"]
    got = [torch.empty(n, dtype=torch.float64, device=DEV) for _ in range(2)]
    alt = torch.empty(n, k, dtype=torch.float64, device=DEV)
    for a in range(0, n, 64):
        lp = torch.log_softmax(d["logits"][a:a + 64].double(), -1)
        got[0][a:a + 64] = lp.gather(1, d["tokens"][a:a + 64, None])[:, 0]
        got[1][a:a + 64] = -(lp.exp() * lp).sum(1)
        alt[a:a + 64] = lp.topk(k, dim=1).values
    return dict(logprob=got[0], entropy=got[1], rank=None, top_tokens=None, top_logprobs=alt)


def exact(case, seed):
    d = _inputs(case, seed)
    return {"evict": _exact_evict, "logp": _exact_logp}.get(case["op"], _exact_attention)(d)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    if case["op"] == "logp":
        n, vocab, k = case["rows"], case["vocab"], case["top"]
        size = 4 if case["dtype"] == "float32" else 2
        return dict(bytes=n * (vocab * size + 8 + 12 + 12 * k), flops=8 * n * vocab)
    rec = _record_bytes(case["dim"], case["group"]) / BLOCK * case["hkv"]       # bytes of a token in a layer
    if case["op"] == "evict":
        n = [case["hi"]] + [(case["lo"] + case["hi"]) / 2] * (case["rows"] - 1)
        kept = sum(case["keep"] if x > case["keep"] else 0 for x in n)
        read = sum(x for x in n if x > case["keep"])
        return dict(bytes=case["layers"] * (kept * (2 * rec + 4) + read * 4), flops=case["layers"] * read)
    rows, m, hq, dim = case["rows"], case["m"], case["hq"], case["dim"]
    ragged = rows > 1 and (case["lo"] < case["hi"] or case["hi"] == 0)
    new = 0.75 * m if ragged else m
    before = (case["lo"] + case["hi"]) / 2
    if case["lo"] == case["hi"] and case["hi"] > m:
        before -= m
    pairs = rows * hq * new * (before + (new + 1) / 2)
    tokens = rows * (before + new)
    if case["op"] == "chunk":
        return dict(bytes=tokens * rec + 4 * rows * hq * new * dim, flops=4 * dim * pairs)
    return dict(bytes=tokens * (rec / 2 + 8) + rows * hq * new * (2 * dim + 4), flops=2 * dim * pairs)
