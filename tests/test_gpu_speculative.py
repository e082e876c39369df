"""GPU: the operators of the 4-bit cache together, as the speculative-decoding example runs them."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    path = os.path.join(ROOT, "adaptive-kv-memory_b200", "examples", "speculative_decode.py")
    spec = importlib.util.spec_from_file_location("speculative_decode", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_greedy_output_is_the_targets_own():
    """At temperature 0 every kept token is the target's best one: fed the finished sequences token by token, the
    target finds it within 2 % of the logits' spread of its maximum (bf16 activations, other tile shapes), and
    nearly always the maximum itself."""
    ex = _example()
    target = ex.Decoder()
    prompts = torch.randint(0, target.vocab, (3, 41), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    tokens, accepted, cache = ex.speculative_generate(target, target.first(3), prompts, n=2, steps=6, k=3, temperature=0)
    R, L = 6, 41
    assert accepted.shape == (6, R) and int(accepted.min()) >= 0 and int(accepted.max()) <= 3
    seqs = [row[row >= 0] for row in tokens]
    lens = [len(s) for s in seqs]
    # everything but the last token is in the cache
    assert cache.lens.tolist() == [n - 1 for n in lens]
    assert lens == [L + 6 + int(a) for a in accepted.sum(0)]
    for a, b in zip(seqs[0::2], seqs[1::2]):  # both continuations of a prompt are the same greedy one
        m = min(len(a), len(b))
        assert torch.equal(a[:m], b[:m])
    c = target.cache(1, 200, 16)
    row = torch.zeros(1, dtype=torch.int32, device="cuda")
    best = 0
    total = 0
    for s in seqs[::2]:
        c.free(row)
        logits = target.forward(s[None, :L], c, row)[0, -1:]
        for t in range(L, len(s)):
            gap = float(logits.max() - logits[0, s[t]])
            assert gap <= 0.02 * float(logits.max() - logits.min()), (t, gap)
            best += gap == 0
            total += 1
            logits = target.forward(s[None, t:t + 1], c, row)[0]
    assert best >= 0.9 * total
    c.check()


def test_sampled_run_keeps_tables_consistent():
    ex = _example()
    target = ex.Decoder(layers=2)
    prompts = torch.randint(0, target.vocab, (2, 33), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    tokens, accepted, cache = ex.speculative_generate(target, target.first(1), prompts, n=3, steps=5, k=2)
    assert int(accepted.sum()) > 0
    used = cache.table[cache.table >= 0]
    counts = torch.bincount(used.long(), minlength=cache.n_pages)
    assert torch.equal(counts.int(), cache.refs)
    # the prompt's full first page is held by all three continuations of its prompt
    assert sorted(cache.refs[cache.table[:, 0].long()].tolist()) == [3] * 6
    before = [cache.read(0, 40, [r], start=[0]) for r in range(6)]
    cache.free([1, 4])
    live = int(cache.compact())
    assert live == int((cache.refs > 0).sum()) and int(cache.refs[:live].min()) >= 1
    cache.check()
    for r in (0, 2, 3, 5):
        k, v = cache.read(0, 40, [r], start=[0])
        assert torch.equal(k, before[r][0]) and torch.equal(v, before[r][1])
