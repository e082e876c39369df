"""Measured cases of the speculative-serving operators over the 4-bit paged cache.

Four operators, each reached as a serving program reaches it:

* ``attend``  attention of 1..n query tokens per sequence over a paged cache held in 4 bits
* ``append``  new K / V rows quantised into the pages, and the values the cache now stands for read back
* ``verify``  acceptance of drafted tokens against the target's probabilities, and the token after them
* ``pages``   forking sequences, reserving pages (copy on write), rolling back, freeing, compacting

``own`` False runs their plain form (elementary torch operations in 32 bits), True the framework's kernels.

The cache: page p of layer l holds, for each KV head, a record of 32 tokens: K codes [32][D/2] bytes (channel 2j in the
high nibble of byte j), V codes [32][D/2], then (scale, zero) fp16 pairs of K [32][G][2] and of V [32][G][2], with
G = D / group.  A code c of a group stands for c * scale + zero.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one conversation on a small model (12 query / 2 KV heads), a 4K context, one token at a time: latency
        dict(name="attend_one_4k", op="attend", rows=1, hq=12, hkv=2, dim=128, group=128, m=1, lo=4096, hi=4096,
             dtype="float16"),
        # a full batch of long contexts, one token each: the ordinary decode step of an 8B-class model's layer
        dict(name="attend_batch_32k", op="attend", rows=16, hq=32, hkv=8, dim=128, group=128, m=1, lo=32768, hi=32768,
             dtype="float16"),
        # the same model scoring four drafted tokens and the one before them, fine groups of 32 channels, odd lengths
        dict(name="attend_draft_32k", op="attend", rows=16, hq=32, hkv=8, dim=128, group=32, m=5, lo=32001, hi=32767,
             dtype="bfloat16"),
        # continuous batching: 64 sequences of 1K to 30K tokens, each with its own number of drafted tokens
        dict(name="attend_ragged_64", op="attend", rows=64, hq=32, hkv=8, dim=128, group=64, m=4, lo=1024, hi=30720,
             dtype="float16"),
        # a decode step's new tokens (64 sequences, up to 5 each) entering the cache
        dict(name="append_step_64", op="append", rows=64, hkv=8, dim=128, group=128, m=5, lo=100, hi=4000,
             dtype="float16"),
        # four prompts of 32K tokens entering the cache at once
        dict(name="append_prompt_32k", op="append", rows=4, hkv=8, dim=128, group=32, m=32767, lo=0, hi=0,
             dtype="bfloat16"),
        # one conversation, four drafted tokens, the vocabulary of the 12 / 2-head model
        dict(name="verify_one", op="verify", rows=1, k=4, vocab=151936, dtype="float32", draft=True),
        # a batch of 64 with up to seven drafts each
        dict(name="verify_batch_64", op="verify", rows=64, k=7, vocab=151936, dtype="float32", draft=True),
        # drafts looked up in the prompt (no draft distribution), probabilities kept in bf16, odd vocabulary
        dict(name="verify_lookup_bf16", op="verify", rows=33, k=3, vocab=32003, dtype="bfloat16", draft=False),
        # best-of-four on one prompt: four continuations share its pages and each copies the partial last one
        dict(name="pages_branch_4", op="pages", kind="branch", layers=2, n_pages=256, hkv=2, dim=128, group=128,
             parents=1, children=4, m=5, lo=3001, hi=3001),
        # best-of-eight on 32 prompts of a 16-layer pool
        dict(name="pages_branch_256", op="pages", kind="branch", layers=16, n_pages=2048, hkv=8, dim=128, group=128,
             parents=32, children=8, m=5, lo=500, hi=1500),
        # half of the sequences have ended: the live pages move to the low end of the pool
        dict(name="pages_compact", op="pages", kind="compact", layers=4, n_pages=8192, hkv=8, dim=128, group=128,
             parents=64, children=0, m=0, lo=500, hi=3600),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "verify", "verify", "pages"])
    if op == "attend":
        dim = rng.choice([64, 128, 128, 256])
        group = rng.choice([g for g in (32, 64, 128, 256) if dim // 4 <= g <= dim])
        hkv = _spread(rng, 1, 8)
        hq = hkv * _spread(rng, 1, 8)
        rows = _spread(rng, 1, 96)
        m = _spread(rng, 1, 12)
        # no more cache than 16 rows of 32K tokens x 8 heads of 128, no more products than the largest listed case
        most = min(65536, 16 * 32768 * 8 * 128 // (rows * hkv * dim), 10 ** 10 // (rows * hq * m * dim))
        hi = _spread(rng, min(16, most), most)
        lo = rng.choice([0, hi, hi // 3])
        return dict(op=op, rows=rows, hq=hq, hkv=hkv, dim=dim, group=group, m=m, lo=lo, hi=hi,
                    dtype=rng.choice(["float16", "bfloat16"]))
    if op == "append":
        dim = rng.choice([64, 128, 128, 256])
        group = rng.choice([g for g in (32, 64, 128, 256) if dim // 4 <= g <= dim])
        hkv, rows = _spread(rng, 1, 8), _spread(rng, 1, 64)
        m = _spread(rng, 1, 4 * 32767 * 8 * 128 // (rows * hkv * dim) // 2 if rows > 4 else 20000)
        hi = _spread(rng, 1, 4000)
        return dict(op=op, rows=rows, hkv=hkv, dim=dim, group=group, m=m, lo=rng.choice([0, hi]), hi=hi,
                    dtype=rng.choice(["float16", "bfloat16"]))
    if op == "verify":
        return dict(op=op, rows=_spread(rng, 1, 64), k=_spread(rng, 1, 8), vocab=_spread(rng, 1000, 152000),
                    dtype=rng.choice(["float32", "float32", "float16", "bfloat16"]), draft=rng.random() < 0.7)
    kind = rng.choice(["branch", "compact"])
    dim = rng.choice([64, 128, 256])
    group = rng.choice([g for g in (32, 64, 128, 256) if dim // 4 <= g <= dim])
    parents = _spread(rng, 1, 32)
    children = _spread(rng, 1, 8) if kind == "branch" else 0
    lo, hi = 40, _spread(rng, 64, 1500)
    n_pages = parents * (hi // BLOCK + 2) * (3 if kind == "compact" else 1) + parents * (1 + children) * 3 + 8
    return dict(op=op, kind=kind, layers=_spread(rng, 1, 4), n_pages=n_pages, hkv=_spread(rng, 1, 8), dim=dim,
                group=group, parents=parents, children=children, m=_spread(rng, 1, 40) if children else 0, lo=lo, hi=hi)


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


def _quantise(x, group):
    """Codes (…, D) int, scale and zero (…, G) fp16 of rows x (…, D): the cache's definition in fp32."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504.0, 65504.0)
    g = x.unflatten(-1, (-1, group))
    lo = g.amin(-1).half()
    s = ((g.amax(-1) - lo.float()) / 15.0).half()
    sf = s.float().unsqueeze(-1)
    q = torch.where(sf > 0, (g - lo.float().unsqueeze(-1)) / sf, torch.zeros_like(g))
    return q.round().clamp(0, 15).flatten(-2).to(torch.uint8), s, lo


def _pack(codes):
    return (codes[..., 0::2] << 4) | codes[..., 1::2]


def _kv_rows(shape, g, dtype):
    """K and V rows as a model makes them: unit normal, a few channels of K several times larger."""
    k = torch.randn(shape, generator=g, device=DEV)
    k[..., 3] *= 6
    k[..., shape[-1] // 2 + 1] *= 4
    v = torch.randn(shape, generator=g, device=DEV)
    return k.to(dtype), v.to(dtype)


def _fields(buf, dim, group):
    """Views of a (…, rec) uint8 buffer: K codes, V codes (…, 32, D/2), K and V (scale, zero) (…, 32, G, 2) fp16."""
    h, n = BLOCK * dim // 2, BLOCK * (dim // group) * 4
    lead = buf.shape[:-1]
    kc = buf[..., :h].unflatten(-1, (BLOCK, dim // 2))
    vc = buf[..., h:2 * h].unflatten(-1, (BLOCK, dim // 2))
    kp = buf[..., 2 * h:2 * h + n].view(torch.float16).unflatten(-1, (BLOCK, dim // group, 2))
    vp = buf[..., 2 * h + n:].view(torch.float16).unflatten(-1, (BLOCK, dim // group, 2))
    assert kc.shape[:-2] == lead
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


def _fill(buf, table, lens, dim, group, g):
    """Quantised K / V of every row written into its pages of layer 0."""
    hkv = buf.shape[2]
    for r, n in enumerate(lens):
        nb = -(-n // BLOCK)
        if nb == 0:
            continue
        pages = table[r, :nb].to(DEV).long()
        rec = torch.empty(nb, hkv, buf.shape[3], dtype=torch.uint8, device=DEV)
        kc, vc, kp, vp = _fields(rec, dim, group)
        for x, c, p in zip(_kv_rows((nb, hkv, BLOCK, dim), g, torch.float16), (kc, vc), (kp, vp)):
            code, s, z = _quantise(x, group)
            c.copy_(_pack(code))
            p[..., 0] = s
            p[..., 1] = z
        buf[0, pages] = rec


def _seq_lens(case, g):
    n = case["rows"]
    lens = _ints(case["lo"], case["hi"], n, g).tolist()
    if n > 3 and case["lo"] < case["hi"]:
        lens[1] = case["hi"]
        lens[2] = case["lo"]
    return lens


def _inputs(case, seed):
    """The case's data, from the seed alone (plain tensors; no handle of the framework)."""
    g, hg = _gen(seed), _host(seed)
    op = case["op"]
    if op == "verify":
        return _verify_inputs(case, g, hg)
    if op == "pages":
        return _pages_inputs(case, g, hg)
    dt = getattr(torch, case["dtype"])
    rows, m, hkv, dim, group = case["rows"], case["m"], case["hkv"], case["dim"], case["group"]
    if op == "attend":
        # lengths after the new tokens; each row scores between 1 and m of them
        lens = _seq_lens(case, hg)
        new = [m] * rows if rows == 1 or case["lo"] == case["hi"] else _ints(1, m, rows, hg).tolist()
        lens = [max(a, b) for a, b in zip(lens, new)]
    else:
        new = [m] * rows if rows <= 4 else _ints(max(1, m // 2), m, rows, hg).tolist()
        lens = [a + b for a, b in zip(_seq_lens(case, hg), new)]
    max_blocks = max(1, max(-(-n // BLOCK) for n in lens))
    n_pages = sum(-(-n // BLOCK) for n in lens) + 3
    table = _tables(lens, n_pages, max_blocks, hg)
    buf = torch.zeros(1, n_pages, hkv, _record_bytes(dim, group), dtype=torch.uint8, device=DEV)
    d = dict(op=op, buf=buf, table=table.to(DEV), lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
             new=torch.tensor(new, dtype=torch.int32, device=DEV), lens_host=lens, new_host=new, dim=dim, group=group,
             dtype=dt, m=m, hkv=hkv)
    if op == "attend":
        _fill(buf, table, lens, dim, group, g)
        # the layout a projection gives: token-major, seen head-major
        d["q"] = torch.randn(rows, m, case["hq"], dim, generator=g, device=DEV).to(dt).transpose(1, 2)
    else:
        k, v = _kv_rows((rows, m, hkv, dim), g, dt)
        d["k"], d["v"] = k.transpose(1, 2), v.transpose(1, 2)
    return d


def _verify_inputs(case, g, hg):
    b, k, vocab = case["rows"], case["k"], case["vocab"]
    dt = getattr(torch, case["dtype"])
    target = torch.empty(b, k + 1, vocab, dtype=dt, device=DEV)
    draft = torch.empty(b, k, vocab, dtype=dt, device=DEV) if case["draft"] else None
    tokens = torch.empty(b, k, dtype=torch.int64, device=DEV)
    for r in range(b):
        # next-token distributions of a model at temperature 1, and a draft model near it
        logits = torch.randn(k + 1, vocab, generator=g, device=DEV) * 3.0
        target[r] = torch.softmax(logits, -1).to(dt)
        q = torch.softmax(logits[:k] + torch.randn(k, vocab, generator=g, device=DEV) * 0.5, -1)
        if draft is not None:
            draft[r] = q.to(dt)
        noise = torch.rand(k, vocab, generator=g, device=DEV).clamp_min(1e-30)
        tokens[r] = (q.log() - (-noise.log()).log()).argmax(-1)
    n = _ints(0, k, b, hg) if b > 1 else torch.tensor([k])
    return dict(op="verify", target=target, draft=draft, tokens=tokens, n_draft=n.int().to(DEV),
                u=torch.rand(b, k, generator=g, device=DEV), u_last=torch.rand(b, generator=g, device=DEV))


def _pages_inputs(case, g, hg):
    parents, children = case["parents"], case["children"]
    lens = _ints(case["lo"], case["hi"], parents, hg).tolist()
    if case["kind"] == "compact":
        # every second sequence has ended and left its pages behind
        used = [-(-n // BLOCK) for n in lens]
        while sum(used) > case["n_pages"] * 3 // 4:
            lens = [max(1, n * 3 // 4) for n in lens]
            used = [-(-n // BLOCK) for n in lens]
    max_seqs = parents * (1 + children) + (2 if case["kind"] == "compact" else 0)
    max_blocks = -(-(case["hi"] + max(case["m"], 1)) // BLOCK)
    table = torch.full((max_seqs, max_blocks), -1, dtype=torch.int32)
    table[:parents] = _tables(lens, case["n_pages"], max_blocks, hg)
    all_lens = torch.zeros(max_seqs, dtype=torch.int32)
    all_lens[:parents] = torch.tensor(lens, dtype=torch.int32)
    if case["kind"] == "compact":
        dead = list(range(1, parents, 2))
        table[dead] = -1
        all_lens[dead] = 0
        # a fork shares its parent's pages
        table[parents] = table[0]
        all_lens[parents] = all_lens[0]
    rec = _record_bytes(case["dim"], case["group"])
    buf = torch.randint(0, 256, (case["layers"], case["n_pages"], case["hkv"], rec), generator=g, device=DEV,
                        dtype=torch.uint8)
    d = dict(op="pages", kind=case["kind"], buf=buf, table=table.to(DEV), lens=all_lens.to(DEV), dim=case["dim"],
             group=case["group"], hkv=case["hkv"], parents=parents, children=children, m=case["m"])
    if case["kind"] == "branch":
        par = torch.arange(parents, dtype=torch.int32).repeat_interleave(children)
        kid = torch.arange(parents, parents * (1 + children), dtype=torch.int32)
        rows = torch.cat([kid, torch.arange(parents, dtype=torch.int32)])
        d.update(par=par.to(DEV), kid=kid.to(DEV), rows_all=rows.to(DEV),
                 new=torch.randint(1, case["m"] + 1, (rows.numel(),), generator=hg, dtype=torch.int32).to(DEV),
                 par_rows=torch.arange(parents, dtype=torch.int32, device=DEV),
                 par_lens=all_lens[:parents].clone().to(DEV))
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    d["own"] = own
    if d["op"] == "pages" or not own:
        d["refs"] = _count_refs(d["table"], d["buf"].shape[1]) if d["op"] == "pages" else None
    if d["op"] == "pages" and d["kind"] == "compact":
        d.update(table0=d["table"].clone(), refs0=d["refs"].clone())
    if not own or d["op"] == "verify":
        return d
    akv = _akv()
    table = d["table"]
    cache = akv.Int4PagedCache(d["buf"].shape[0], d["buf"].shape[1], d["hkv"], d["dim"], group_size=d["group"],
                               max_seqs=table.shape[0], max_blocks=table.shape[1], device=DEV)
    cache.load_state(d.pop("buf"), d["table"], d["lens"])
    d["cache"] = cache
    if d["op"] == "pages" and d["kind"] == "compact":
        d["state0"] = cache.page_state()
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
    return {"attend": _plain_attend, "append": _plain_append, "verify": _plain_verify,
            "pages": _plain_pages}[state["op"]](state)


def _run_own(s):
    op = s["op"]
    if op == "verify":
        n, tokens = _akv().verify_draft(s["target"], s["draft"], s["tokens"], s["u"], s["u_last"],
                                        n_draft=s["n_draft"])
        return dict(accepted=n, tokens=tokens)
    c = s["cache"]
    if op == "attend":
        out, lse = c.attend(0, s["q"], n_new=s["new"], return_lse=True)
        return dict(out=out, lse=lse)
    if op == "append":
        c.append(0, s["k"], s["v"], n_new=s["new"])
        k, v = c.read(0, s["m"], n_new=s["new"], dtype=s["dtype"])
        return dict(k=k, v=v)
    if s["kind"] == "compact":
        c.set_page_state(s["state0"])
        live = c.compact()
        return dict(live=live, table=c.table, lens=c.lens, refs=c.refs, buf=c.buf)
    c.fork(s["par"], s["kid"])
    granted = c.reserve(s["rows_all"], s["new"])
    table, lens, refs = c.table.clone(), c.lens.clone(), c.refs.clone()
    c.free(s["kid"])
    c.truncate(s["par_rows"], s["par_lens"])
    return dict(granted=granted, table=table, lens=lens, refs=refs, table_after=c.table, refs_after=c.refs, buf=c.buf)


# ------------------------------------------------------------------------------------------------ plain forms
def _values(codes, pairs, group):
    """fp32 values (…, D) of codes (…, D/2) bytes and (scale, zero) pairs (…, G, 2)."""
    c = torch.stack([codes >> 4, codes & 15], -1).flatten(-2).float().unflatten(-1, (-1, group))
    return (c * pairs[..., 0:1].float() + pairs[..., 1:2].float()).flatten(-2)


def _plain_attend(s):
    rows, hq, m, dim = s["q"].shape
    hkv, group = s["hkv"], s["group"]
    rep = hq // hkv
    rec = s["buf"][0, s["table"].clamp_min(0).long()].transpose(1, 2)      # (rows, hkv, blocks, rec)
    kc, vc, kp, vp = _fields(rec, dim, group)
    q = s["q"].float().unflatten(1, (hkv, rep)).flatten(2, 3)              # (rows, hkv, rep * m, D)
    x = (q @ _values(kc, kp, group).flatten(2, 3).transpose(2, 3)).unflatten(2, (rep, m)) / math.sqrt(dim)
    i = torch.arange(m, device=q.device)
    t = torch.arange(x.shape[-1], device=q.device)
    new, n = s["new"].long(), s["lens"].long()
    seen = (t <= (n - new)[:, None, None] + i[None, :, None]) & (i[None, :] < new[:, None])[:, :, None]
    x = torch.where(seen[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(-3.0e38)
    e = (x - top).exp()
    z = e.sum(-1, keepdim=True)
    w = torch.where(z > 0, e / z, 0.0).flatten(2, 3)
    out = (w @ _values(vc, vp, group).flatten(2, 3)).unflatten(2, (rep, m)).flatten(1, 2)
    lse = torch.where(z > 0, top + z.log(), -math.inf).squeeze(-1).flatten(1, 2)
    return dict(out=out.to(s["dtype"]), lse=lse)


def _plain_append(s):
    rows, hkv, m, dim = s["k"].shape
    group = s["group"]
    back = []
    kc, vc, kp, vp = _fields(s["buf"], dim, group)
    i = torch.arange(m, device=s["k"].device)
    pos = (s["lens"] - s["new"]).long()[:, None] + i[None, :]
    on = i[None, :] < s["new"][:, None]
    block = torch.where(on, pos // BLOCK, 0)
    page = s["table"].long().gather(1, block.clamp_max(s["table"].shape[1] - 1))
    slot = pos % BLOCK
    r, t = on.nonzero(as_tuple=True)
    for x, c, p in ((s["k"], kc, kp), (s["v"], vc, vp)):
        code, sc, z = _quantise(x[r, :, t], group)          # (T, H, D)
        c[0][page[r, t], :, slot[r, t]] = _pack(code)
        p[0][page[r, t], :, slot[r, t]] = torch.stack([sc, z], -1)
        val = _values(c[0][page[r, t], :, slot[r, t]], p[0][page[r, t], :, slot[r, t]], group)
        o = torch.zeros(rows, m, hkv, dim, device=x.device, dtype=s["dtype"])
        o[r, t] = val.to(s["dtype"])
        back.append(o.transpose(1, 2))
    return dict(k=back[0], v=back[1])


def _units(p):
    """Probabilities in whole units of 2^-40."""
    p = torch.nan_to_num(p.float(), nan=0.0, posinf=1.0, neginf=0.0).clamp(0.0, 1.0)
    return (p * 1099511627776.0).round().to(torch.int64)


def _plain_verify(s):
    t, q, x = s["target"], s["draft"], s["tokens"]
    b, k = x.shape
    px = t[:, :k].gather(2, x.unsqueeze(-1)).squeeze(-1).float()
    qx = torch.ones_like(px) if q is None else q.gather(2, x.unsqueeze(-1)).squeeze(-1).float()
    j = torch.arange(k, device=t.device)
    n = s["n_draft"].long()
    ok = (s["u"] * qx < px) & (j[None, :] < n[:, None])
    acc = ok.int().cumprod(1).sum(1).long()
    row = torch.arange(b, device=t.device)
    p_row = _units(t[row, acc])
    at = acc.clamp_max(k - 1)
    if q is None:
        q_row = torch.zeros_like(p_row)
        q_row.scatter_(1, x.gather(1, at[:, None]), 1 << 40)
    else:
        q_row = _units(q[row, at])
    w = torch.where((acc < n)[:, None], (p_row - q_row).clamp_min(0), p_row)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, p_row)
    total = w.sum(1)
    u24 = (s["u_last"] * 16777216.0).floor().to(torch.int64)
    goal = (total >> 24) * u24 + (((total & 0xFFFFFF) * u24) >> 24)
    last = (w.cumsum(1) <= goal[:, None]).sum(1)
    last = torch.where(total > 0, last, -1)
    out = torch.where(torch.arange(k + 1, device=t.device)[None, :] < acc[:, None],
                      torch.cat([x, x[:, :1]], 1), -1)
    out.scatter_(1, acc[:, None], last[:, None])
    return dict(accepted=acc.int(), tokens=out)


def _drop(table, refs, lens, rows, new_lens):
    """Rows shortened to new_lens: their pages beyond it given back."""
    rows = rows.long()
    j = torch.arange(table.shape[1], device=table.device)
    t = table[rows]
    gone = (j[None, :] >= ((new_lens + BLOCK - 1) // BLOCK)[:, None]) & (t >= 0)
    refs.index_add_(0, torch.where(gone, t, 0).flatten().long(), -gone.flatten().to(refs.dtype))
    table[rows] = torch.where(gone, -1, t)
    lens[rows] = new_lens


def _plain_pages(s):
    table, lens, refs, buf = s["table"], s["lens"], s["refs"], s["buf"]
    if s["kind"] == "compact":
        table.copy_(s["table0"])
        refs.copy_(s["refs0"])
        live = refs > 0
        n_live = live.sum()
        i = torch.arange(refs.numel(), device=refs.device)
        holes = (~live & (i < n_live)).nonzero().squeeze(1)
        movers = (live & (i >= n_live)).nonzero().squeeze(1)
        to = i.clone()
        to[movers] = holes
        table.copy_(torch.where(table >= 0, to[table.clamp_min(0).long()].int(), table))
        buf[:, holes] = buf[:, movers]
        refs[holes] = refs[movers]
        refs[movers] = 0
        return dict(live=n_live.int().reshape(1), table=table, lens=lens, refs=refs, buf=buf)
    par, kid = s["par"].long(), s["kid"].long()
    # fork: the children see the parents' pages
    table[kid] = table[par]
    lens[kid] = lens[par]
    t = table[kid]
    refs.index_add_(0, t.clamp_min(0).flatten().long(), (t >= 0).flatten().to(refs.dtype))
    # reserve: new pages for the new tokens, and a page of its own for a row that would write into a shared one
    rows, new = s["rows_all"].long(), s["new"]
    n0 = lens[rows]
    nb0, nb1 = (n0 + BLOCK - 1) // BLOCK, (n0 + new + BLOCK - 1) // BLOCK
    part = (n0 % BLOCK != 0) & (new > 0)
    last = table[rows, (nb0 - 1).clamp_min(0).long()].long()
    same = (last[:, None] == last[None, :]) & part[None, :] & part[:, None]
    before = torch.tril(same, -1).sum(1)
    cow = part & (refs[last.clamp_min(0)] - before > 1)
    need = (nb1 - nb0) + cow.int()
    off = need.cumsum(0) - need
    free = torch.argsort((refs > 0).int(), stable=True)       # the free pages first, lowest index first
    w = int(need.max())
    slot = torch.arange(w, device=table.device)[None, :]
    on = slot < need[:, None]
    r, c = on.nonzero(as_tuple=True)
    page = free[off[r] + c]
    refs[page] = 1
    block = nb0[r] - cow[r].int() + c
    src = last[cow]
    table[rows[r], block.long()] = page.int()
    buf[:, free[off[cow].long()]] = buf[:, src]
    refs.index_add_(0, src, torch.full_like(src, -1).to(refs.dtype))
    lens[rows] = n0 + new
    mid = table.clone(), lens.clone(), refs.clone()
    _drop(table, refs, lens, s["kid"], torch.zeros_like(s["kid"]))
    _drop(table, refs, lens, s["par_rows"], s["par_lens"])
    return dict(granted=new.clone(), table=mid[0], lens=mid[1], refs=mid[2], table_after=table, refs_after=refs, buf=buf)


# ------------------------------------------------------------------------------------------------ the least a pass moves
def work(case):
    op = case["op"]
    if op == "verify":
        size = {"float32": 4, "float16": 2, "bfloat16": 2}[case["dtype"]]
        rows = case["rows"] * case["vocab"]
        reads = 2 if case["draft"] else 1
        return dict(bytes=rows * reads * size + case["rows"] * case["k"] * 32, flops=rows * (reads + 2))
    if op == "pages":
        page = case["hkv"] * _record_bytes(case["dim"], case["group"])
        avg = (case["lo"] + case["hi"]) / 2
        if case["kind"] == "branch":
            copied = case["parents"] * case["children"] * case["layers"]
            entries = case["parents"] * (1 + case["children"]) * avg / BLOCK
        else:
            live = min(case["parents"] * avg / BLOCK, case["n_pages"] * 0.75) / 2
            copied = live * (1 - live / case["n_pages"]) * case["layers"]
            entries = live
        return dict(bytes=int(2 * copied * page + 16 * entries), flops=int(entries))
    rec = case["hkv"] * (case["dim"] + 8 * (case["dim"] // case["group"]))
    if op == "append":
        new = case["rows"] * (case["m"] if case["rows"] <= 4 else case["m"] * 0.75)
        half = 4 * case["hkv"] * case["dim"]
        # rows in, records out, records in, values out
        return dict(bytes=int(new * (2 * half + 2 * rec)), flops=int(new * case["hkv"] * case["dim"] * 2 * 8))
    avg = max((case["lo"] + case["hi"]) / 2, 1)
    new = case["m"] if case["rows"] == 1 or case["lo"] == case["hi"] else (1 + case["m"]) / 2
    io = case["rows"] * case["hq"] * new * case["dim"] * 4
    return dict(bytes=int(case["rows"] * avg * rec + io),
                flops=int(4 * case["rows"] * avg * case["hq"] * new * case["dim"]))


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    d = _inputs(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "verify": _exact_verify,
            "pages": lambda d, c: None}[d["op"]](d, case)


def _wide(codes, pairs, group):
    """codes (…, D/2) bytes and (…, G, 2) pairs to (…, D) in 64 bits."""
    hi, lo = (codes // 16).double(), (codes % 16).double()
    dim = codes.shape[-1] * 2
    v = torch.empty(*codes.shape[:-1], dim, dtype=torch.float64, device=codes.device)
    v[..., 0::2] = hi
    v[..., 1::2] = lo
    sc = pairs[..., 0].double().repeat_interleave(group, -1)
    ze = pairs[..., 1].double().repeat_interleave(group, -1)
    return v * sc + ze


def _exact_attend(d, case):
    q = d["q"].double()
    rows, hq, m, dim = q.shape
    rep = hq // d["hkv"]
    out = torch.zeros(rows, hq, m, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((rows, hq, m), -math.inf, dtype=torch.float64, device=q.device)
    table = d["table"].long()
    kc, vc, kp, vp = _fields(d["buf"][0], dim, d["group"])
    for r in range(rows):
        n, new = d["lens_host"][r], d["new_host"][r]
        pages = table[r, :-(-n // BLOCK)]
        for h in range(d["hkv"]):
            k = _wide(kc[pages, h], kp[pages, h], d["group"]).reshape(-1, dim)[:n]
            v = _wide(vc[pages, h], vp[pages, h], d["group"]).reshape(-1, dim)[:n]
            for i in range(new):
                end = n - new + i + 1
                logit = q[r, h * rep:(h + 1) * rep, i] @ k[:end].T / math.sqrt(dim)
                lse[r, h * rep:(h + 1) * rep, i] = torch.logsumexp(logit, -1)
                out[r, h * rep:(h + 1) * rep, i] = torch.softmax(logit, -1) @ v[:end]
    return dict(out=out, lse=lse)


def _exact_append(d, case):
    res = {}
    keep = torch.arange(d["m"], device=DEV)[None, :] < d["new"][:, None]
    for name in ("k", "v"):
        x = d[name].transpose(1, 2).double()                 # (rows, m, H, D)
        shape = x.shape
        x = x.reshape(*shape[:-1], shape[-1] // d["group"], d["group"])
        lo = x.min(-1, keepdim=True).values                   # a value of the input: exact in fp16 when that is its type
        lo = lo.to(torch.float16).double()
        step = ((x.max(-1, keepdim=True).values - lo) / 15).to(torch.float16).double()
        code = torch.round((x - lo) / step.clamp_min(1e-30)).clamp_(0, 15)
        val = (code * step + lo).reshape(shape)
        val[~keep] = 0
        res[name] = val.transpose(1, 2)
        del x, code
    return res


def _exact_verify(d, case):
    import numpy as np
    t = d["target"]
    b, k1, vocab = t.shape
    x, u = d["tokens"].cpu().numpy(), d["u"].double().cpu().numpy()
    n, ul = d["n_draft"].cpu().numpy(), d["u_last"].double().cpu().numpy()
    accepted = np.zeros(b, np.int32)
    tokens = np.full((b, k1), -1, np.int64)
    for r in range(b):
        j = 0
        while j < n[r]:
            p = float(t[r, j, x[r, j]])
            q = 1.0 if d["draft"] is None else float(d["draft"][r, j, x[r, j]])
            if not u[r, j] * q < p:
                break
            tokens[r, j] = x[r, j]
            j += 1
        accepted[r] = j
        full = np.rint(np.clip(t[r, j].double().cpu().numpy(), 0, 1) * 2.0 ** 40).astype(np.int64)
        w = full
        if j < n[r]:
            w = full.copy()
            if d["draft"] is None:
                w[x[r, j]] = 0
            else:
                w -= np.rint(np.clip(d["draft"][r, j].double().cpu().numpy(), 0, 1) * 2.0 ** 40).astype(np.int64)
                w[w < 0] = 0
            if w.sum() == 0:
                w = full
        total = int(w.sum())
        if total:
            goal = int(ul[r] * 2 ** 24) * total >> 24
            tokens[r, j] = int(np.searchsorted(np.cumsum(w), goal, side="right"))
    return dict(accepted=torch.from_numpy(accepted), tokens=torch.from_numpy(tokens))
