"""GPU: attention weight where (tokens x query heads of a group) passes 32 bits: the oldest tokens count too."""
import pytest
import torch

from test_gpu_int4_weigh import DEV, _cache, _query

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,rep,group", [(700_001, 4096, 64), (700_001, 4096, 16), (300_000, 4096, 64)])
def test_old_tokens_of_many_heads(n, rep, group):
    """Tolerance as in test_gpu_int4_weigh.py, with |x| and the bound taken at their largest over the tokens looked at:
    x is off by 2^-20 B + 2^-22 (B + |x| + |lse|) + 2^-21, B the sum of |q| |K| / 8 over the channels; 2^-24 * 4,224 of
    the sum for adding rep terms (128 at a time) one by one."""
    blocks = -(-n // 32)
    c = _cache(pages=blocks, heads=1, dim=64, group=group, seqs=1, blocks=blocks)
    granted = c.reserve([0], n)
    k = torch.randn(1, 1, n, 64, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).half()
    c.append(0, k, k, None, granted)
    c.check()
    q = _query((1, rep, 1, 64), 3, torch.bfloat16)
    lse = torch.full((1, rep, 1), 9.0, device=DEV)
    c.weigh(0, q, lse)
    c.check()
    for at in (0, 1000, n // 2, n - 40):
        stored, _ = c.read(0, 40, None, torch.tensor([at], dtype=torch.int32, device=DEV), dtype=torch.float16)
        kd, qd = stored[0, 0].double(), q[0, :, 0].double()
        # read() rounds c*s + z to fp16: 2^-11 of a value, one more term of x's error
        x = qd @ kd.T / 8
        b = qd.abs() @ (kd.abs() + 1.0) .T / 8
        off = (2.0 ** -20 + 2.0 ** -22 + 2.0 ** -11) * 2 * b + 2.0 ** -22 * (x.abs() + 9) + 2.0 ** -21
        e = (x - 9).exp()
        want, tol = e.sum(0), (e * off).sum(0) * 1.1 + 2.0 ** -24 * 4224 * e.sum(0)
        assert ((c.weights[0, 0, at:at + 40].double() - want).abs() <= tol).all(), at
