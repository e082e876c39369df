"""GPU: eviction of as many rows as a call takes, and the refusal of more."""
import pytest
import torch

from test_gpu_int4_weigh import DEV, _cache

pytestmark = pytest.mark.gpu


def test_most_rows_of_a_call():
    n = 65536
    c = _cache(pages=64, heads=1, dim=64, seqs=n, blocks=1)
    rows = torch.tensor([0, 40000, n - 1], dtype=torch.int32, device=DEV)
    k = torch.randn(3, 1, 20, 64, device=DEV).half()
    c.append(0, k, k, rows, c.reserve(rows, 20))
    c.weights[0, :, :20] = torch.arange(20, device=DEV).float()
    state = c.page_state()
    with pytest.raises(ValueError, match="65535"):
        c.evict(None, 7)
    assert torch.equal(c.page_state(), state)
    kept = c.evict(torch.arange(n - 1, 0, -1, dtype=torch.int32, device=DEV), 7, first=2)
    c.check()
    want = torch.tensor([0, 1, 15, 16, 17, 18, 19], dtype=torch.int32, device=DEV)
    held = torch.tensor([0, n - 1 - 40000], device=DEV)      # where the rows with tokens stand in the call
    assert (kept[held] == want).all()
    others = torch.ones(n - 1, dtype=torch.bool, device=DEV)
    others[held] = False
    assert (kept[others] == -1).all()
    assert c.lens[rows.long()].tolist() == [20, 7, 7] and int(c.lens.sum()) == 34
