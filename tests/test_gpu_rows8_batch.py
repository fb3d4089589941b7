"""What of a token's norm does not depend on how many tokens share the call, and what does."""
import pytest
import torch

from tropical_gemm import rows8
from tropical_gemm.rows8 import Rows8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# rows on both sides of two and of four times the number of SMs, where the norm changes its shape and its kernel
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [128, 1000, 1111, 4096, 8192])
def test_a_row_alone_and_among_others(dtype, cols):
    """h and its 8-bit checkpoint are the same bits: maxima are exact.  The sum of squares may be taken in another order, so
    the factor and the norm's scale differ by twice the bound of one sum (at most 64 terms in a thread and 64 sums joined, half of
    it through the root, and 6 roundings), and a code next to a tie may be the neighbour."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    x, res = (torch.randn(2000, cols, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = torch.randn(cols, generator=g, device="cuda").to(dtype)
    whole = rows8.rmsnorm(x, w, residual=res, checkpoint=True)
    again = rows8.rmsnorm(x, w, residual=res, checkpoint=True)
    for s, t in ((whole.rows.q, again.rows.q), (whole.rows.scale, again.rows.scale), (whole.rstd, again.rstd)):
        assert torch.equal(s, t)   # the same call: the same bits
    for rows in (1, 16, 296, 300, 592, 600):
        n = rows8.rmsnorm(x[:rows], w, residual=res[:rows], checkpoint=True)
        assert torch.equal(n.h, whole.h[:rows])
        assert torch.equal(n.checkpoint.q, whole.checkpoint.q[:rows]) and torch.equal(n.checkpoint.scale, whole.checkpoint.scale[:rows])
        rel = 2 * (0.5 * 128 + 6) * U
        assert ((n.rstd - whole.rstd[:rows]).abs() <= whole.rstd[:rows] * rel).all()
        assert ((n.rows.scale - whole.rows.scale[:rows]).abs() <= whole.rows.scale[:rows] * rel).all()
        off = (n.rows.q.to(torch.int16) - whole.rows.q[:rows].to(torch.int16)).abs()
        # a code changes where the quotient, 127 at most, comes within its own change, 127 * (rel + 4 U) < 2^-9, of a tie
        assert off.max() <= 1 and off.sum() <= max(8, off.numel() * 2.0 ** -8)
        # the product's bits depend on the 8-bit rows alone
        b = Rows8(whole.rows.q[:64], whole.rows.scale[:64])
        z = rows8.matmul(n.rows, b, dtype=dtype)
        assert torch.equal(z, rows8.matmul(Rows8(torch.cat([n.rows.q, whole.rows.q]), torch.cat([n.rows.scale, whole.rows.scale])), b, dtype=dtype)[:rows])
