"""GPU: device-side page ownership against a host model (fork, reserve with copy on write, truncate, free, compact).

The model keeps lists: every table entry, length, reference count and page byte has to match exactly after every
operation of long random sequences.
"""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


class Model:
    def __init__(self, layers, pages, seqs, blocks, content):
        self.pages, self.blocks = pages, blocks
        self.rows = [[] for _ in range(seqs)]
        self.lens = [0] * seqs
        self.content = content.copy()  # page -> what it holds

    def refs(self):
        r = [0] * self.pages
        for row in self.rows:
            for p in row:
                r[p] += 1
        return r

    def fork(self, parents, children):
        for i, (p, c) in enumerate(zip(parents, children)):
            if p in children or c in children[:i] or self.lens[c]:
                continue
            self.rows[c], self.lens[c] = list(self.rows[p]), self.lens[p]

    def reserve(self, rows, n_new):
        refs, granted, done, copies = self.refs(), [], False, []
        free = [p for p in range(self.pages) if refs[p] == 0]
        for i, (r, n) in enumerate(zip(rows, n_new)):
            nb0, nb1 = -(-self.lens[r] // 32), -(-(self.lens[r] + n) // 32)
            if r in rows[:i] or nb1 > self.blocks or n < 0:
                granted.append(0)
                continue
            part = n > 0 and self.lens[r] % 32 != 0
            cow = part and refs[self.rows[r][-1]] > 1
            if done or nb1 - nb0 + cow > len(free):
                done = True
                granted.append(0)
                continue
            if cow:
                p = free.pop(0)
                refs[self.rows[r][-1]] -= 1
                copies.append((self.rows[r][-1], p))
                self.rows[r][-1] = p
            for _ in range(nb1 - nb0):
                self.rows[r].append(free.pop(0))
            self.lens[r] += n
            granted.append(n)
        for a, b in copies:
            self.content[b] = self.content[a]
        return granted

    def truncate(self, rows, new):
        for i, (r, n) in enumerate(zip(rows, new)):
            if r in rows[:i] or not 0 <= n <= self.lens[r]:
                continue
            self.rows[r], self.lens[r] = self.rows[r][:-(-n // 32)], n

    def compact(self):
        refs = self.refs()
        live = sum(x > 0 for x in refs)
        holes = [p for p in range(live) if refs[p] == 0]
        movers = [p for p in range(live, self.pages) if refs[p]]
        to = dict(zip(movers, holes))
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]
        for a, b in to.items():
            self.content[b] = self.content[a]
        return live


def _same(c, m, content):
    c_table, refs = c.table.cpu().tolist(), m.refs()
    assert c.lens.tolist() == m.lens
    assert [[p for p in row if p >= 0] for row in c_table] == m.rows
    assert all(p == -1 for row, mr in zip(c_table, m.rows) for p in row[len(mr):])
    assert c.refs.tolist() == refs
    bits = c.free_bits.cpu().numpy().view("uint32")
    free = [(int(bits[p // 32]) >> (p % 32)) & 1 for p in range(len(bits) * 32)]
    assert free == [int(p < c.n_pages and refs[p] == 0) for p in range(len(bits) * 32)]
    idx = torch.tensor([m.content[p] for p in range(c.n_pages)])
    assert torch.equal(c.buf.cpu(), content[:, idx])


def _make(layers=2, pages=50, seqs=9, blocks=6, heads=1, dim=64):
    import akv
    c = akv.Int4PagedCache(layers, pages, heads, dim, max_seqs=seqs, max_blocks=blocks, device=DEV)
    c.buf.random_(0, 256)
    content = c.buf.cpu().clone()
    return c, Model(layers, pages, seqs, blocks, {p: p for p in range(pages)}), content


@pytest.mark.parametrize("seed,pages", [(0, 50), (1, 20), (2, 33), (3, 400)])
def test_random_histories(seed, pages):
    rng = random.Random(seed)
    c, m, content = _make(pages=pages)
    seqs, cap = 9, 6 * 32
    for step in range(60):
        op = rng.choice(["reserve", "reserve", "fork", "truncate", "free", "compact"])
        rows = rng.sample(range(seqs), rng.randint(1, seqs))
        if op == "reserve":
            n = [rng.choice([0, 1, 5, 31, 32, 33, 64, 200]) for _ in rows]
            if rng.random() < 0.1:
                rows[-1] = rows[0]
            assert c.reserve(rows, n).tolist() == m.reserve(rows, n)
        elif op == "fork":
            half = len(rows) // 2
            par, kid = [rng.choice(range(seqs)) for _ in range(half)], rows[:half]
            c.fork(par, kid)
            m.fork(par, kid)
        elif op == "truncate":
            n = [rng.choice([m.lens[r], m.lens[r] // 2, max(0, m.lens[r] - 1), 0, cap + 1]) for r in rows]
            c.truncate(rows, torch.tensor(n, dtype=torch.int32, device=DEV))
            m.truncate(rows, n)
        elif op == "free":
            c.free(rows[:2])
            m.truncate(rows[:2], [0, 0])
        else:
            assert int(c.compact()) == m.compact()
        c.status.zero_()
        _same(c, m, content)


def test_copy_on_write_in_request_order():
    """Three holders of a partly filled page: the first two to write copy it, the last keeps it."""
    c, m, content = _make()
    for x in (c, m):
        x.reserve([0], [40])
        x.fork([0, 0], [1, 2])
    assert c.refs.tolist()[:3] == [3, 3, 0]
    assert c.reserve([2, 0, 1], [1, 1, 1]).tolist() == m.reserve([2, 0, 1], [1, 1, 1]) == [1, 1, 1]
    c.check()
    _same(c, m, content)
    assert [c.table[r, 1].item() for r in (2, 0, 1)] == [2, 3, 1]


def test_exhausted_pool_refuses_in_order():
    c, m, content = _make(pages=4)
    assert c.reserve([0, 1, 2, 3], [64, 64, 32, 0]).tolist() == m.reserve([0, 1, 2, 3], [64, 64, 32, 0]) == [64, 64, 0, 0]
    with pytest.raises(RuntimeError, match="AKV_ERR_EXHAUSTED"):
        c.check()
    c.check()  # cleared
    _same(c, m, content)
    # refused rows write and see nothing
    k = torch.ones(4, 1, 2, 64, dtype=torch.float16, device=DEV)
    before = c.buf.clone()
    g = c.reserve([2], 1)
    c.append(0, k[:1], k[:1], [2], g)
    assert torch.equal(c.buf, before)
    assert (c.attend(0, k[:1], [2], g) == 0).all()


def test_many_requests_and_pages():
    """More requests than one plan holds, and more pages than one scan of the free bits."""
    import akv
    c = akv.Int4PagedCache(1, 40000, 1, 64, max_seqs=1500, max_blocks=30, device=DEV)
    assert c.reserve(None, 800).tolist() == [800] * 1500
    c.check()
    assert torch.equal(c.table[:, :25], torch.arange(37500, dtype=torch.int32, device=DEV).view(1500, 25))
    odd = torch.arange(1, 1500, 2, dtype=torch.int32, device=DEV)
    c.free(odd)
    assert int(c.compact()) == 750 * 25
    c.check()
    assert int(c.refs[:18750].min()) == 1 and int(c.refs[18750:].max()) == 0
    assert c.free_pages() == 40000 - 18750
    live = c.table[0::2, :25]
    assert torch.equal(live.flatten().sort().values, torch.arange(18750, dtype=torch.int32, device=DEV))


def test_copy_pages_and_refusals():
    import akv
    c, m, content = _make(layers=3, heads=3, dim=256)
    src, dst = [1, 7, 3], [2, 9, 4]
    c.copy_pages(src, dst)
    c.check()
    want = content.clone()
    want[:, dst] = content[:, src]
    assert torch.equal(c.buf.cpu(), want)
    c.copy_pages([0], [50])
    with pytest.raises(RuntimeError, match="AKV_ERR_SHAPE"):
        c.check()
    assert torch.equal(c.buf.cpu(), want)
    for call in (lambda: c.reserve([0, 99], 1), lambda: c.fork([0], [0]), lambda: c.truncate([0], [5]),
                 lambda: c.reserve([0], 32 * 7), lambda: c.free([-1])):
        call()
        with pytest.raises(RuntimeError, match="AKV_ERR_SHAPE"):
            c.check()
    with pytest.raises(ValueError):
        c.reserve([0], -1)
    with pytest.raises(ValueError):
        c.fork([0, 1], [2])
    with pytest.raises(ValueError):
        c.truncate([0, 1], [2])
    c.reserve([], 1)
    c.fork([], [])
    c.check()
    assert isinstance(akv.Int4PagedCache, type)
