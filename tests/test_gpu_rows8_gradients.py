"""Gradients of the 8-bit product on the GPU, held to the size of their results: the 2-norm of the error over the 2-norm
of the 64-bit result, which a missing or doubled term of a long sum shows in, as a worst-case bound does not."""
import pytest
import torch

from tropical_gemm import rows8
from tropical_gemm.rows8 import Rows8

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def rand8(g, rows, cols, dtype):
    """8-bit rows; for bf16 gradients with scales that are powers of two, so that the values, rounded to bf16 on
    their way to the tensor core, are exact and what is left is the sums' error."""
    scale = torch.rand(rows, generator=g, device="cuda") * 0.02 + 1e-3
    if dtype == torch.bfloat16:
        scale = torch.exp2(torch.floor(torch.log2(scale)))
    return Rows8(torch.randint(-127, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int8), scale)


def error(got, want):
    return float((got.double() - want).norm() / want.norm())


def values(r):
    return r.q.double() * r.scale.double()[:, None]


# outputs p x c of sums of r terms: parts of the sum in several pairs, one tile at a time, two tiles at a time
LONG = [(8, 24, 2_000_003), (130, 200, 300_000), (2048, 1280, 70_001), (4864, 4352, 20_000)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("p, c, r", LONG)
@pytest.mark.parametrize("rows", [True, False])
def test_sums_of_16_bit_gradients_keep_16_bits_at_any_length(dtype, p, c, r, rows):
    """The tensor core loses 1e-9 of a sum per term (1.5e-5 after 16384 terms of bf16; f16 8e-6 after 8192, beside 4.9e-6
    of 16 carried bits), so sums are added up in f32 after so many: twice that is the bound."""
    g = gen(p + r)
    b, grad = rand8(g, r, c, dtype), randn(g, *((p, r) if rows else (r, p)), dtype=dtype)
    ga, gb = rows8.matmul_backward(grad, None if rows else b, b if rows else None, dtype_a=torch.float32, dtype_b=torch.float32)
    want = (grad.double() if rows else grad.double().t()) @ values(b)
    assert error(ga if rows else gb, want) < 2.0 ** -15
