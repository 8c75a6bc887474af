"""Root-mean-square norm: calls whose offsets pass 32 bits."""
import pytest
import torch

import fairseq_apollo_b200 as M


@pytest.mark.gpu
@pytest.mark.parametrize("dim,groups", [(2048, 1), (2048, 16), (2041, 1)])
def test_more_than_2_to_the_31_values(dim, groups):
    """the last rows of a long call, forward and backward, against a call of their own; the weight's gradient over all rows"""
    rows, tail = 2 ** 31 // dim + 1000, 700
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    g = torch.Generator(device="cuda").manual_seed(0)
    x, res, dy, dr = (torch.randn(1, rows, dim, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(4))
    assert x.numel() > 2 ** 31
    weight = (torch.randn(dim, device="cuda", generator=g) * 0.1).requires_grad_()

    def call(x, res, dy, dr):
        x, res = x.detach().requires_grad_(), res.detach().requires_grad_()
        y, r = M.rms_norm(x, weight, res, groups)
        dx, dw = torch.autograd.grad([y, r], [x, weight], [dy, dr])
        return y.detach(), r.detach(), dx, dw
    whole = call(x, res, dy, dr)
    last = call(*(t[:, -tail:].contiguous() for t in (x, res, dy, dr)))
    for a, b in zip(whole[:3], last[:3]):
        assert torch.equal(a[:, -tail:], b)   # (a row is one warp's or one block's in both)
    # the weight's gradient is the sum of the pieces': sums of 2^20 terms of size 1 in fp32, in another order
    want = torch.zeros(dim, dtype=torch.float64, device="cuda")
    for part in range(0, rows, rows // 4 + 1):
        cut = slice(part, min(rows, part + rows // 4 + 1))
        want += call(*(t[:, cut] for t in (x, res, dy, dr)))[3].double()
    # (each row's term is dy r / rms, about 1 in size: partial sums stay below 2^13, and a sum has rows / 8 / 296 + 300 additions at most)
    assert float((whole[3].double() - want).abs().max()) < 2 * (rows / 2368 + 300) * 2.0 ** -24 * 2 ** 13
