"""GPU: chunk attention, weights, eviction and token log probabilities together, as a bounded cache uses them.

Each step's tolerance is the operator's own, from its tests; what an eviction leaves is compared byte for byte."""
import importlib.util
import math
import os

import pytest
import test_gpu_int4_chunk as chunk
import test_gpu_int4_evict as evict
import test_gpu_int4_weigh as weigh
import test_gpu_token_logprobs as logprobs
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"


@pytest.mark.parametrize("dim,group,rep,dtype", [(64, 32, 3, torch.bfloat16), (128, 128, 4, torch.float16)])
def test_chunks_then_tokens(dim, group, rep, dtype):
    import akv
    c = akv.Int4PagedCache(2, 64, 2, dim, group_size=group, max_seqs=4, max_blocks=16, device=DEV, track_weights=True)
    g = torch.Generator(device=DEV).manual_seed(dim)
    rows = [2, 0, 3]
    r = evict._i(*rows)
    head = torch.randn(2 * rep * dim, 700, generator=g, device=DEV)
    for step, new in enumerate(([150, 70, 0], [150, 33, 64], [90, 150, 1], [1, 1, 1], [1, 0, 1])):
        M = max(new)
        granted = c.reserve(r, evict._i(*new))
        assert granted.tolist() == new
        for layer in range(2):
            k, v = (torch.randn(3, 2, M, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
            q = torch.randn(3, 2 * rep, M, dim, generator=g, device=DEV).to(dtype)
            c.append(layer, k, v, r, granted)
            out, lse = (c.attend if M == 1 else c.attend_chunk)(layer, q, r, granted, return_lse=True)
            if M > 1:
                chunk._check(c, q, out, lse, rows, new, layer)
            before = c.weights.clone()
            c.weigh(layer, q, lse, r, granted)
            weigh._check(c, before, weigh._expected(c, layer, q, lse, rows, new), layer)
            # each query's weights sum to 1: the lse's tolerance is below 1e-3, fp32 sums are far below it
            got = (c.weights[layer].double() - before[layer].double()).sum(1)[torch.tensor(rows, device=DEV)]
            want = torch.tensor(new, device=DEV) * 2.0 * rep
            assert ((got - want).abs() <= 1e-3 * want + 2.0 ** -20 * before[layer].double().sum()).all()
        logits = (out.transpose(1, 2).reshape(3 * M, -1).float() @ head).to(dtype)
        tokens = torch.randint(0, 700, (3 * M,), generator=g, device=DEV)
        logprobs._check(logits, tokens, akv.token_logprobs(logits, tokens, top=3), 3)
        evict._run(c, rows, 120, first=4, recent=20)
        assert int(c.lens.max()) <= 120
    c.check()
    assert int((c.refs > 0).sum()) == sum(math.ceil(n / 32) for n in c.lens.tolist())


def test_example_runs():
    path = os.path.join(ROOT, "adaptive-kv-memory_b200", "examples", "bounded_context.py")
    spec = importlib.util.spec_from_file_location("bounded_context", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    model = ex.BoundedDecoder(layers=2)
    g = torch.Generator("cuda").manual_seed(5)
    lengths = torch.tensor([300, 65, 130], device="cuda")
    texts = torch.randint(0, model.vocab, (3, 300), device="cuda", generator=g)
    scored, new, cache = ex.score(model, texts, lengths, chunk=64, keep=96, first=2, recent=16, more=5)
    assert scored.logprob.shape == scored.entropy.shape == scored.rank.shape == (3, 299)
    inside = torch.arange(1, 300, device="cuda")[None] < lengths[:, None]
    assert torch.isfinite(scored.logprob[inside]).all() and (scored.logprob[inside] <= 0).all()
    assert scored.logprob[~inside].isnan().all() and (scored.rank[~inside] == 0).all()
    assert (scored.rank[inside] >= 1).all() and (scored.rank[inside] <= model.vocab).all()
    assert new.shape == (3, 5) and int(new.min()) >= 0 and int(new.max()) < model.vocab
    assert cache.lens.tolist() == [96, 70, 96]
    used = cache.table[cache.table >= 0]
    assert torch.equal(torch.bincount(used.long(), minlength=cache.n_pages).int(), cache.refs)


def test_calls_on_several_streams_at_once():
    """Chunks, weights, evictions and log probabilities of three caches side by side: the results of one after another."""
    import akv

    def work(seed):
        c = akv.Int4PagedCache(2, 80, 2, 64, group_size=32, max_seqs=4, max_blocks=20, device=DEV, track_weights=True)
        weigh._fill(c, [600, 333, 500], seed)
        rows = evict._i(0, 1, 2)
        q = weigh._query((3, 8, 300, 64), seed, torch.bfloat16)
        logits = weigh._query((300, 30001), seed, torch.bfloat16)
        torch.cuda.synchronize()
        out = []

        def run():
            for _ in range(5):
                o, lse = c.attend_chunk(0, q, rows, return_lse=True)
                c.weigh(0, q, lse, rows)
                c.weigh(1, q[:, :, -2:], lse[:, :, -2:], rows)
                out.append((o, c.weights.clone(), akv.token_logprobs(logits, torch.zeros(300, dtype=torch.int64, device=DEV),
                                                                     top=4).top_logprobs))
            out.append((c.evict(rows, 200, 4, 50), c.weights, c.lens, c.table, c.buf))
        return run, out, c
    alone = [work(s) for s in range(3)]
    for run, _, c in alone:
        run()
        c.check()
    beside = [work(s) for s in range(3)]
    streams = [torch.cuda.Stream() for _ in beside]
    for (run, _, _), s in zip(beside, streams):
        with torch.cuda.stream(s):
            run()
    torch.cuda.synchronize()
    for (_, a, _), (_, b, c) in zip(alone, beside):
        c.check()
        for x, y in zip(a, b):
            assert all(torch.equal(p, q) for p, q in zip(x, y))
