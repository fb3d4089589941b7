"""8-bit products on the GPU where one kernel gives way to another: the same bits on both sides."""
import pytest
import torch

from tropical_gemm import rows8
from tropical_gemm.rows8 import Rows8

pytestmark = pytest.mark.gpu


def rand8(g, rows, cols):
    return Rows8(torch.randint(-127, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int8),
                 torch.rand(rows, generator=g, device="cuda") * 0.02 + 1e-3)


# channels around 15 and 33 tiles of 128 (clusters that run at once), and around half as many tiles as SMs
@pytest.mark.parametrize("n", [1920, 1928, 2304, 2400, 4224, 4232, 4736, 4800, 9472, 9480])
@pytest.mark.parametrize("k", [640, 4112])
def test_bits_are_the_same_on_both_sides_of_a_choice(n, k):
    g = torch.Generator(device="cuda").manual_seed(n + k)
    a, b = rand8(g, 520, k), rand8(g, n, k)
    bias = torch.randn(n, generator=g, device="cuda")
    whole = rows8.matmul(a, b, bias=bias, dtype=torch.float32)   # 520 tokens: the paired kernel
    # integer sums below 2^26 are exact in 64-bit floats; then three roundings of 2^-24 at most
    want = (a.q.double() @ b.q.double().t()) * a.scale.double()[:, None] * b.scale.double()
    off = (whole.double() - want - bias.double()).abs()
    assert (off <= want.abs() * 2.0 ** -22 + (want + bias.double()).abs() * 2.0 ** -23).all()
    for m in (1, 16, 33, 64, 65, 128, 129, 256, 384, 512):
        assert torch.equal(rows8.matmul(Rows8(a.q[:m], a.scale[:m]), b, bias=bias, dtype=torch.float32), whole[:m])
