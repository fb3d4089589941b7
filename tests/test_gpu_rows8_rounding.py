"""Rounding to 8 bits on the GPU: q is x / scale rounded to nearest even, in every kernel that quantises."""
import pytest
import torch

from tropical_gemm import rows8

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def check_codes(q, x):
    """`q` against x * 127 / max|x| rounded to nearest even, without a rounding on the way: for values of at most 24
    bits 127 |x| and q max|x| have 31, so they and their difference are exact in 64-bit floats (or q is 0 and the
    difference is 127 |x| itself).  Exact ties have to go to even.  Others may go to either side of a tie that the f32
    quotient does not tell from them: it is off by 127 * 2^-23 at most, 2 R by twice that, below 2^-15, of top; rows
    whose max|x| / 127 is exact round it to units of 2^-15 first, another 2^-16 off: 2 R by less than 2^-14 top."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    mag = x.abs() * 127
    low = torch.floor(mag / top)
    low = torch.where(mag - low * top < 0, low - 1, low)   # the division rounds: the remainder is in [0, top)
    low = torch.where(mag - low * top >= top, low + 1, low)
    rest = 2 * (mag - low * top)
    want = torch.where((rest > top) | ((rest == top) & (low % 2 == 1)), low + 1, low) * x.sign()
    exact = (top / 127).float().double() * 127 == top
    free = (rest != top) & ((rest - top).abs() <= top * torch.where(exact, 2.0 ** -14, 2.0 ** -15))
    off = (q.double() - want).abs()
    assert not ((off != 0) & ~free).any(), f"{int(((off != 0) & ~free).sum())} codes off, {int((rest == top).sum())} ties"
    assert (off <= 1).all()
    return int((rest == top).sum())


def half_steps(rows, cols, step, dtype, seed):
    """Rows of multiples of step / 2, exact in `dtype`, whose largest magnitude is 127 steps: full of ties."""
    x = torch.randint(-254, 255, (rows, cols), generator=gen(seed), device="cuda").double() * (step / 2)
    x[:, -1] = 127 * step
    y = x.to(dtype)
    keep = y.double() == x
    keep[:, -1] = True
    y = torch.where(keep, y, torch.zeros_like(y))
    assert (y[:, -1].double() == 127 * step).all()
    return y


def test_a_row_of_ties():
    x = torch.tensor([[381, 1.5, 7.5, 13.5, -1.5, -7.5, 4.5, -10.5]], device="cuda")
    assert rows8.quantize(x).q.tolist() == [[127, 0, 2, 4, 0, -2, 2, -4]]


# odd multiples of 127 that the type holds (bf16, of 8 bits, holds 127 itself only), and powers of two
STEPS = {torch.float32: [1.0, 3.0, 5.0, 7.0 * 2.0 ** -40, 1001.0 * 2.0 ** 30, 131071.0, 3.0 * 2.0 ** -126],
         torch.float16: [1.0, 3.0, 5.0, 15.0, 11.0 * 2.0 ** -14], torch.bfloat16: [1.0, 2.0 ** -100]}
# one row per block and per warp, long rows, rows that start anywhere, rows off all boundaries
SHAPES = [(1, 8, 0), (3, 17, 0), (5, 256, 0), (700, 1024, 0), (2, 8192, 0), (2, 16391, 0), (3, 33000, 0), (40, 61, 3), (6, 512, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols, first", SHAPES)
def test_quantize_ties_go_to_even(dtype, rows, cols, first):
    ties = 0
    for i, step in enumerate(STEPS[dtype]):
        wide = torch.zeros(rows, cols + first, device="cuda", dtype=dtype)
        wide[:, first:] = half_steps(rows, cols, step, dtype, i)
        ties += check_codes(rows8.quantize(wide[:, first:]).q, wide[:, first:])
    assert ties or dtype != torch.float32


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols, first", SHAPES)
@pytest.mark.parametrize("step", [1.0, 3.0, 5.0, 11.0])
def test_checkpoint_ties_go_to_even(dtype, rows, cols, first, step):
    """The checkpoint of h = x + residual, where the largest magnitude has more bits than the type."""
    h = half_steps(rows, cols, step, torch.float32, rows)
    x = torch.zeros(rows, cols + first, device="cuda", dtype=dtype)
    x[:, first:] = h.to(dtype)
    res = torch.zeros_like(x)
    res[:, first:] = (h - x[:, first:].float()).to(dtype)
    x, res = x[:, first:], res[:, first:]
    assert torch.equal(x.float() + res.float(), h)
    n = rows8.rmsnorm(x, torch.ones(cols, device="cuda", dtype=dtype), residual=res, checkpoint=True)
    assert check_codes(n.checkpoint.q, h) > 0 or cols <= 17


def row_of_mean_square(mean, head, cols):
    """A row of integers that starts with `head` and whose squares add up to mean * cols exactly."""
    row, left = list(head), int(mean) * cols - sum(v * v for v in head)
    while len(row) < cols - 4:
        v = int((left / (cols - len(row))) ** 0.5)
        row.append(v)
        left -= v * v
    for a in range(int(left ** 0.5), -1, -1):   # every number is a sum of four squares
        for b in range(int((left - a * a) ** 0.5), -1, -1):
            for c in range(int((left - a * a - b * b) ** 0.5), -1, -1):
                d = left - a * a - b * b - c * c
                if int(d ** 0.5 + 0.5) ** 2 == d:
                    return row + [a, b, c, int(d ** 0.5 + 0.5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows", [1, 300, 2000])
@pytest.mark.parametrize("first", [0, 3])
def test_norm_ties_go_to_even(dtype, rows, first):
    """A row whose root mean square is 256: every sum of squares on the way is an integer of at most 24 bits and the norm
    of h is h / 256, so its ties are those of h (762 = 127 * 6, and 6 (n + 1/2) with either sign)."""
    h = torch.tensor(row_of_mean_square(2 ** 16, [762, 3, 15, 27, -3, -15, 9, -21], 256), device="cuda", dtype=torch.float64)
    assert h.square().sum() == 2 ** 24 and h.abs().max() == 762
    wide = torch.zeros(rows, 256 + first, device="cuda", dtype=dtype)
    wide[:, first:] = h.to(dtype)
    n = rows8.rmsnorm(wide[:, first:], torch.ones(256, device="cuda", dtype=dtype), eps=0.0, checkpoint=True)
    assert (n.rstd == 1 / 256).all()
    assert check_codes(n.rows.q, h.expand(rows, 256)) >= 7 * rows
    assert check_codes(n.checkpoint.q, h.expand(rows, 256)) >= 7 * rows


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", [(4, 9), (200, 999), (800, 4096), (40, 16390)])
def test_random_rows(dtype, rows, cols):
    x = torch.randn(rows, cols, generator=gen(cols), device="cuda").to(dtype)
    x[::5] *= 2.0 ** -20 if dtype != torch.float16 else 1.0
    check_codes(rows8.quantize(x).q, x)
    res = torch.randn(rows, cols, generator=gen(rows), device="cuda").to(dtype)
    n = rows8.rmsnorm(x, torch.ones(cols, device="cuda", dtype=dtype), residual=res, checkpoint=True)
    check_codes(n.checkpoint.q, x.float() + res.float())
