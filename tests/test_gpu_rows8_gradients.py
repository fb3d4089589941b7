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


# outputs p x c of sums of r terms, f32: one tile and few blocks; sums in parts with chunks in each; several tiles per
# pair with chunks, whole and ragged edges; narrow outputs
F32 = [(512, 256, 512), (300, 200, 5000), (24, 8, 200_000), (2100, 4100, 4100), (2048, 4096, 1024), (3000, 100, 8191), (513, 1025, 1087)]


@pytest.mark.parametrize("p, c, r", F32)
@pytest.mark.parametrize("rows", [True, False])
def test_f32_gradients_are_f32(p, c, r, rows):
    """A product of f32 operands in f32 would lose 4e-7 to 2.5e-6 here.  This one carries all 24 bits of g and lets the tensor
    core add 1024 terms at most, which loses 6.6e-7.  Without the chunks 4100 terms lose 2.9e-6, without the third
    part of g every sum 4.9e-6."""
    g = gen(p + c)
    b, grad = rand8(g, r, c, torch.float32), randn(g, *((p, r) if rows else (r, p)))
    ga, gb = rows8.matmul_backward(grad, None if rows else b, b if rows else None)
    want = (grad.double() if rows else grad.double().t()) @ values(b)
    assert error(ga if rows else gb, want) < 1e-6


# p x c outputs of r terms where pairs take two tiles at a time (more than 74 couples of 256-row tiles): an even and an odd
# number of row tiles, single tiles after the doubles, ragged edges, rings that wrap (11 blocks and more) and a short sum
DOUBLE = [(4700, 4300, 700), (5000, 4097, 64), (4864, 4096, 1000), (7200, 2600, 1337), (40000, 200, 390)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("p, c, r", DOUBLE)
@pytest.mark.parametrize("rows", [True, False])
def test_gradients_two_tiles_at_a_time(dtype, p, c, r, rows):
    """Errors as above: factors of 16 bits (f16: 4.9e-6 at random) or exact (bf16 with scales of powers of two), and sums
    that lose 1e-9 per term, 2e-6 at most here; a tile that is wrong, missing or in another's place shows at once.  Each tile is
    held to the bound too, its own error over its own size."""
    g = gen(p + c + r)
    b, grad = rand8(g, r, c, dtype), randn(g, *((p, r) if rows else (r, p)), dtype=dtype)
    ga, gb = rows8.matmul_backward(grad, None if rows else b, b if rows else None, dtype_a=torch.float32, dtype_b=torch.float32)
    got = (ga if rows else gb).double()
    want = (grad.double() if rows else grad.double().t()) @ values(b)
    bound = 2.0 ** -16
    assert error(got, want) < bound
    pad = (0, -c % 256, 0, -p % 256)
    tiles = [torch.nn.functional.pad(v, pad).square().unflatten(0, (-1, 256)).unflatten(2, (-1, 256)).sum((1, 3)) for v in (got - want, want)]
    assert (tiles[0] <= bound ** 2 * tiles[1]).all()
    ga, gb = rows8.matmul_backward(grad, None if rows else b, b if rows else None)   # and in its own type
    assert torch.equal(ga if rows else gb, got.to(dtype))
