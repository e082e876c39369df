"""GPU: more than 1,024 requests in one reserve call, against the host model of the page operations.

The plan takes 1,024 requests at a time; its answer has to be that of one list: refused from the first request that
the pool cannot serve, a repeated row refused, shared pages left in request order.
"""
import random

import pytest
import torch

import test_gpu_page_table as base

pytestmark = pytest.mark.gpu


def _status(c):
    code = int(c.status.item())
    c.status.zero_()
    return code


@pytest.mark.parametrize("rows", [None, "list"])
def test_a_pool_that_runs_out_before_the_seam(rows):
    """Page 1,000 is the last: requests 1,000 to 1,499 are refused, those past the seam too."""
    c, m, content = base._make(layers=1, pages=1000, seqs=1500, blocks=2)
    ask = list(range(1500))
    want = m.reserve(ask, [20] * 1500)
    assert want == [20] * 1000 + [0] * 500
    got = c.reserve(None if rows is None else ask, 20)
    assert got.tolist() == want
    assert _status(c) == -9
    base._same(c, m, content)


def test_one_large_request_refuses_all_after_it():
    """The pool still has pages for what follows the refused request, before and after the seam."""
    c, m, content = base._make(layers=1, pages=1225, seqs=1300, blocks=9)
    n = [10 if i < 700 or i % 3 else 0 for i in range(1300)]
    for i in range(560, 600):
        n[i] = 288                                       # nine pages each
    n[1000] = 288
    ask = list(range(1300))
    random.Random(1).shuffle(ask)
    want = m.reserve(ask, n)
    assert any(want[990:1000]) and not any(want[1000:])  # nine pages wanted, five left
    assert c.reserve(ask, torch.tensor(n, dtype=torch.int32, device=base.DEV)).tolist() == want
    assert _status(c) == -9
    base._same(c, m, content)


def test_rows_repeated_across_the_seam():
    c, m, content = base._make(layers=1, pages=3000, seqs=1400, blocks=3)
    ask = list(range(1400))
    ask[1100], ask[1101], ask[1399], ask[3] = 7, 1023, 1023, 9
    n = [(7 * i) % 60 for i in range(1400)]
    assert c.reserve(ask, n).tolist() == m.reserve(ask, n)
    assert _status(c) == -1
    base._same(c, m, content)
    assert c.lens[7].item() == n[7] and c.lens[1023].item() == n[1023]


def test_a_repeated_row_whose_first_request_was_refused():
    c, m, content = base._make(layers=1, pages=300, seqs=20, blocks=3)
    assert c.reserve([4, 4, 5], [97, 10, 10]).tolist() == m.reserve([4, 4, 5], [97, 10, 10]) == [0, 0, 10]
    assert _status(c) == -1
    base._same(c, m, content)


def test_one_page_shared_by_rows_on_both_sides_of_the_seam():
    """1,200 continuations of one prompt: all but the last to be asked for copy its partly filled page."""
    c, m, content = base._make(layers=2, pages=1300, seqs=1201, blocks=3)
    c.reserve([5], [40])
    m.reserve([5], [40])
    kids = [r for r in range(1201) if r != 5]
    c.fork([5] * 1200, kids)
    m.fork([5] * 1200, kids)
    ask = kids[:700] + [5] + kids[700:]
    assert c.reserve(ask, 1).tolist() == m.reserve(ask, [1] * 1201) == [1] * 1201
    assert _status(c) == 0
    base._same(c, m, content)
    assert c.table[ask[-1], 1].item() == 1               # the last one keeps the page


@pytest.mark.parametrize("seed", [0, 1])
def test_random_histories_of_many_rows(seed):
    rng = random.Random(seed)
    seqs = 1300
    c, m, content = base._make(layers=1, pages=2600, seqs=seqs, blocks=5)
    for step in range(12):
        rows = rng.sample(range(seqs), rng.randint(1025, seqs))
        if step % 3 == 0:
            half = len(rows) // 2
            c.free(rows[:half])
            m.truncate(rows[:half], [0] * half)
            par = [rng.choice(rows[half:]) for _ in range(half)]
            c.fork(par, rows[:half])
            m.fork(par, rows[:half])
        n = [rng.choice([0, 1, 5, 31, 33, 70]) for _ in rows]
        for _ in range(rng.randint(0, 3)):
            rows[rng.randrange(len(rows))] = rows[rng.randrange(len(rows))]
        assert c.reserve(rows, n).tolist() == m.reserve(rows, n)
        if step % 4 == 3:
            assert int(c.compact()) == m.compact()
        c.status.zero_()
        base._same(c, m, content)


def test_too_many_requests():
    c, m, content = base._make(pages=50, seqs=9)
    assert c.reserve([0] * 1024, 1).tolist() == [1] + [0] * 1023
    assert _status(c) == -1
    with pytest.raises(ValueError):
        c.reserve([0] * 1025, 1)
    assert c.lens.tolist() == [1] + [0] * 8


def test_free_bits_past_the_pool_are_no_pages():
    """A state whose last word has bits that stand for no page: as many pages are handed out as there are."""
    c, m, content = base._make(layers=1, pages=35, seqs=9, blocks=6)
    c.free_bits.fill_(-1)
    assert c.reserve(list(range(9)), 160).tolist() == m.reserve(list(range(9)), [160] * 9) == [160] * 7 + [0, 0]
    assert _status(c) == -9
    c.free_bits[1] &= 7                                  # what is left of them
    base._same(c, m, content)
