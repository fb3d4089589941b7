"""Layer norm of sums: the gradients of x + residual against their formula in 64 bits.

The sum of two 16-bit numbers has more digits than its type.  y, mean and rstd are of the unrounded sum, and so is the u of the
gradients: nothing but f32 arithmetic and the rounding of each result to its type is allowed for.

With v the f32 sum (half a step of |h|), mean within F32 |mean| + 8 F32 max |h| and rstd within 32 half steps (what the forward
is held to), u is off by at most F32 (10 max |h| rstd + 36 max |u|) < 64 F32 (1 + max |u|) (1 + max |h| rstd / 8).  It stands in
grad_x twice, times rstd max |a| (1 + max |u|), and once in the weight's gradient, times |grad|, where a slot's rows and a join
add at most 64 half steps of each term."""
import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import norms
from _layer_forms import HALF, TINY, TYPES, close, norm, norm_backward

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
# one row; rows loaded directly: whole groups, rows that start anywhere, two groups per thread; from 148 rows on by copies: few columns, odd
# ones, more rows per block than it has stages; too long for registers
SHAPES = [(1, 4096), (5, 8), (33, 200), (9, 1001), (40, 6000), (160, 250), (700, 257), (333, 4096), (2400, 4099), (2400, 8192), (3, 8200), (200, 9001)]


def make(rows, cols, dtype, offset):
    g = torch.Generator(device="cuda").manual_seed(rows * 31 + cols)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    return ((n(rows, cols) + offset).to(dtype), (2 * n(rows, cols)).to(dtype), (1 + 0.2 * n(cols)).to(dtype), (0.2 * n(cols)).to(dtype), n(rows, cols).to(dtype),
            n(rows, cols).to(dtype))


def check(grads, x, res, w, g, gh):
    h, u, rstd, _ = norm(x, res)
    wx, ww, wb = norm_backward(g, u, rstd, w, gh)
    a = (g.double() * (1 if w is None else w.double())).abs().amax(-1, keepdim=True)
    far = 1 + h.abs().amax(-1, keepdim=True) * rstd / 8
    big = 1 + u.abs().amax(-1, keepdim=True)
    half, tiny = 1.01 * HALF[x.dtype], TINY[x.dtype]
    gx, gw, gb = grads
    if gx is not None:
        close(gx, wx, half, 2 * 64 * F32 * rstd * a * big ** 2 * far + (0 if gh is None else 2 * F32 * gh.double().abs()) + tiny)
    if gw is not None:
        close(gw, ww, half, (g.double().abs() * 64 * F32 * (big * far + u.abs())).sum(0) + tiny)
    if gb is not None:
        close(gb, wb, half, 64 * F32 * g.double().abs().sum(0) + tiny)


@pytest.mark.parametrize("offset", [0.0, 50.0])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_autograd(rows, cols, dtype, offset):
    x, res, w, b, g, gh = make(rows, cols, dtype, offset)
    leaves = [t.requires_grad_(True) for t in (x, w, b, res)]
    y, h = tp.layernorm(x, w, b, residual=res)
    gx, gw, gb, gr = torch.autograd.grad((y, h), leaves, (g, gh), retain_graph=True)
    assert torch.equal(gx, gr)
    plain = [t.detach() for t in (x, res, w)]
    check((gx, gw, gb), *plain, g, gh)
    check((*torch.autograd.grad(y, leaves[:3], g, retain_graph=True),), *plain, g, None)
    (only,) = torch.autograd.grad(y, w, g)
    assert torch.equal(only, gw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_calls(rows, cols, dtype):
    """norms.layernorm_backward with the sum's parts: with and without weight and grad_h, run twice, and with rows of wider matrices."""
    x, res, w, b, g, gh = make(rows, cols, dtype, 20.0)
    f = norms.layernorm(x, w, b, residual=res, stats=True)
    for weight, grad_h in ((w, gh), (None, gh), (w, None)):
        got = norms.layernorm_backward(g, x, f.mean, f.rstd, weight, grad_h, residual=res)
        check(got, x, res, weight, g, grad_h)
        again = norms.layernorm_backward(g, x, f.mean, f.rstd, weight, grad_h, residual=res)
        assert all(torch.equal(p, q) for p, q in zip(got, again))
    for skip in (1, 8):
        wide = [torch.full((rows, cols + 17), 7.0, device="cuda", dtype=dtype) for _ in range(2)]
        xs, rs = (t[:, skip:skip + cols] for t in wide)
        xs.copy_(x)
        rs.copy_(res)
        before = [t.clone() for t in wide]
        check(norms.layernorm_backward(g, xs, f.mean, f.rstd, w, gh, residual=rs), x, res, w, g, gh)
        check(norms.layernorm_backward(g, x, f.mean, f.rstd, w, gh, residual=rs), x, res, w, g, gh)
        assert all(torch.equal(s, t) for s, t in zip(wide, before))


@pytest.mark.parametrize("dtype", TYPES)
def test_the_sum_alone(dtype):
    """Without a residual, and with h that is the sum: as before."""
    x, res, w, b, g, gh = make(300, 520, dtype, 3.0)
    f = norms.layernorm(x, w, b, stats=True)
    got = norms.layernorm_backward(g, x, f.mean, f.rstd, w, gh)
    check(got, x, None, w, g, gh)
    zeros = norms.layernorm_backward(g, x, f.mean, f.rstd, w, gh, residual=torch.zeros_like(x))
    for p, q in zip(got, zeros):   # its rows, three operands of a ring, may be joined in another order
        close(p, q.double(), 2 * HALF[dtype], 64 * F32 * float(g.float().abs().sum(0).max()) * 8)
    if dtype == torch.float32:
        s = norms.layernorm(x, w, b, residual=res, stats=True)
        for p, q in zip(norms.layernorm_backward(g, s.h, s.mean, s.rstd, w, gh), norms.layernorm_backward(g, x, s.mean, s.rstd, w, gh, residual=res)):
            close(p, q.double(), 2 * F32, 64 * F32 * float(g.abs().sum(0).max()) * 8)


def test_a_tensor_as_its_own_residual_and_leading_dimensions():
    x, _, w, b, g, gh = make(24, 264, torch.bfloat16, 5.0)
    x3, g3 = x.view(2, 12, 264).transpose(0, 1).requires_grad_(True), g.view(2, 12, 264).transpose(0, 1)
    y, _ = tp.layernorm(x3, w, b, residual=x3)
    (got,) = torch.autograd.grad(y, x3, g3)
    plain = x.detach()
    _, u, rstd, _ = norm(plain, plain)
    want = 2 * norm_backward(g, u, rstd, w)[0]   # two equal gradients, added up in bfloat16
    close(got.transpose(0, 1).reshape(24, 264), want, 3 * HALF[torch.bfloat16], 64 * F32 * float(rstd.max()) * 64)


def test_changed_inputs_are_told():
    x, res, w, b, g, _ = make(6, 64, torch.bfloat16, 0.0)
    w.requires_grad_(True)
    for t in (x, res):
        y, _ = tp.layernorm(x, w, b, residual=res)
        t.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, w, g)


def test_refusals():
    x, res, w, b, g, gh = make(6, 64, torch.bfloat16, 0.0)
    f = norms.layernorm(x, residual=res, stats=True)
    for bad in (res[:, :63], res.float(), res[:5]):
        with pytest.raises(ValueError, match="residual must be like h"):
            norms.layernorm_backward(g, x, f.mean, f.rstd, residual=bad)
    with pytest.raises(ValueError, match="same device"):
        norms.layernorm_backward(g, x, f.mean, f.rstd, residual=res.cpu())
