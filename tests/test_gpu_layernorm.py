"""Layer norm on the GPU, forward and backward, against its formula in 64 bits.

Tolerances count roundings: one to the output's type (half a step), and those of
the f32 arithmetic before it.  f32 sums over `cols` elements in a tree of a few
dozen additions, means and products keep u and y within 32 half steps of f32 of
the row's scale: the row's largest |h - mean| rstd for u."""
import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import blocks8, norms
from _layer_forms import HALF, TINY, TYPES, blocks, close, norm, norm_backward, values

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 8), (2, 128), (17, 129), (300, 1), (129, 130), (31, 1000), (9, 1001), (700, 257), (4, 4095), (1, 8192), (333, 4096),
          (6, 8193), (5, 16384), (3, 16385), (2, 40000), (400, 6000)]


def make(rows, cols, dtype, seed=0, offset=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows * 31 + cols)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    return ((n(rows, cols) + offset).to(dtype), (n(rows, cols) * 2).to(dtype), (1 + 0.2 * n(cols)).to(dtype), (0.2 * n(cols)).to(dtype), n(rows, cols).to(dtype),
            n(rows, cols).to(dtype))


def norm_floor(h, u, rstd, weight, cols):
    """What f32 rounding may change y by: u's error, 32 half steps of the row's largest |u| (and the mean's rounding, of the size of h, times rstd), times weight."""
    size = u.abs().amax(-1, keepdim=True) + 1
    mean = h.abs().amax(-1, keepdim=True) * rstd
    w = 1.0 if weight is None else weight.double().abs()
    return 32 * F32 * (size + mean / 8) * w


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_forward(rows, cols, dtype):
    x, res, w, b, _, _ = make(rows, cols, dtype)
    for residual, weight, bias in ((res, w, b), (None, w, b), (res, None, None), (None, w, None), (None, None, b)):
        r = norms.layernorm(x, weight, bias, residual=residual, stats=True)
        h, u, rstd, y = norm(x, residual, weight, bias)
        close(r.h, h, HALF[dtype], TINY[dtype])
        close(r.y, y, 1.01 * HALF[dtype], norm_floor(h, u, rstd, weight, cols) + 4 * F32 * (0 if bias is None else bias.double().abs()) + TINY[dtype])
        close(r.mean, h.mean(-1), F32, 8 * F32 * h.abs().amax(-1))
        close(r.rstd, rstd[:, 0], 32 * F32 + 16 * F32 * float((h.abs().amax(-1) * rstd[:, 0]).max()))
        again = norms.layernorm(x, weight, bias, residual=residual, stats=True)
        assert torch.equal(r.y, again.y) and torch.equal(r.rstd, again.rstd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_backward(rows, cols, dtype):
    """grad_x = rstd (a - mean a - u mean(a u)) + grad_h: f32 errors of the size of rstd times the row's largest |a| (1 + |u|)."""
    x, _, w, _, g, gh = make(rows, cols, dtype, 1)
    f = norms.layernorm(x, w, None, stats=True)
    h, u, rstd, _ = norm(x)
    for weight, grad_h in ((w, gh), (w, None), (None, gh)):
        gx, gw, gb = norms.layernorm_backward(g, x, f.mean, f.rstd, weight, grad_h)
        wx, ww, wb = norm_backward(g, u, rstd, weight, grad_h)
        a = (g.double() * (1 if weight is None else weight.double())).abs().amax(-1, keepdim=True)
        size = rstd * a * (1 + u.abs().amax(-1, keepdim=True)) ** 2 * (1 + h.abs().amax(-1, keepdim=True) * rstd / 8)
        close(gx, wx, 1.01 * HALF[dtype], 64 * F32 * size + (0 if grad_h is None else 2 * F32 * grad_h.double().abs()) + TINY[dtype])
        # f32 sums over rows: a slot's share in turn, then a join, 64 additions deep at most here; each of a term's size
        each = (g.double().abs() * (u.abs() + h.abs() * rstd)).sum(0)
        close(gw, ww, 1.01 * HALF[dtype], 64 * F32 * (each + (g.double().abs() * (1 + u.abs().amax())).sum(0)) + TINY[dtype])
        close(gb, wb, 1.01 * HALF[dtype], 64 * F32 * g.double().abs().sum(0) + TINY[dtype])
        for p, q in zip((gx, gw, gb), norms.layernorm_backward(g, x, f.mean, f.rstd, weight, grad_h)):
            assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols, pad, skip", [(5, 64, 3, 1), (40, 257, 8, 8), (9, 1000, 5, 2), (600, 130, 2, 6), (3, 9000, 7, 3), (2, 20000, 1, 1)])
def test_strided_rows(rows, cols, pad, skip, dtype):
    """Rows of a wider matrix, from any element on; each operand from another place."""
    wide = [torch.randn(rows, cols + pad + skip + 16, device="cuda").to(dtype) for _ in range(4)]
    x, res, g, gh = (t[:, skip + i:skip + i + cols] for i, t in enumerate(wide))
    w, b = (torch.randn(cols + 1, device="cuda").to(dtype)[1:] for _ in range(2))
    dense = [t.contiguous() for t in (x, res, g, gh, w, b)]
    one, two = norms.layernorm(x, w, b, residual=res, stats=True), norms.layernorm(dense[0], dense[4], dense[5], residual=dense[1], stats=True)
    assert torch.equal(one.h, two.h)
    close(one.y, two.y.double(), 4 * HALF[dtype], 64 * F32 * 8)
    p = norms.layernorm_backward(g, x, one.mean, one.rstd, w, gh)
    q = norms.layernorm_backward(dense[2], dense[0], one.mean, one.rstd, dense[4], dense[3])
    for s, t in zip(p, q):
        close(s, t.double(), 4 * HALF[dtype], 256 * F32 * float(t.abs().max()) + TINY[dtype])
    before = [t.clone() for t in wide]
    assert all(torch.equal(s, t) for s, t in zip(wide, before))


def test_leading_dimensions_and_order():
    x = torch.randn(3, 4, 96, device="cuda")
    w, b = torch.randn(96, device="cuda"), torch.randn(96, device="cuda")
    want = norms.layernorm(x.reshape(12, 96), w, b).y.view(3, 4, 96)
    assert torch.equal(norms.layernorm(x, w, b).y, want)
    turned = x.transpose(0, 1)
    assert torch.equal(norms.layernorm(turned, w, b).y, want.transpose(0, 1))
    columns = torch.randn(96, 7, device="cuda").t()   # elements of a row are not contiguous
    assert torch.equal(norms.layernorm(columns, w, b).y, norms.layernorm(columns.contiguous(), w, b).y)
    one = torch.randn(96, device="cuda")
    assert torch.equal(norms.layernorm(one, w, b).y, norms.layernorm(one[None], w, b).y[0])
    assert norms.layernorm(torch.empty(0, 96, device="cuda"), w, b, stats=True).rstd.shape == (0,)


@pytest.mark.parametrize("cols", [64, 1001, 20000])
def test_large_means_and_constant_rows(cols):
    """A row far from zero: the variance is that of h - mean.  Its f32 inputs hold the spread to 2^-24 of the mean, and so do means."""
    x = torch.randn(8, cols, device="cuda") + 4096.0
    r = norms.layernorm(x, stats=True)
    h, u, rstd, y = norm(x)
    close(r.rstd, rstd[:, 0], 1e-5)   # mean within half a step of 4096 * 2^-24 * 32: (0.5 * 2^-12 * 2^-6)^2 and 32 half steps of f32
    close(r.y, y, F32, 32 * F32 * 8 + 4096 * F32 * 2)
    same = torch.full((4, cols), 3.0, device="cuda")
    b = torch.randn(cols, device="cuda")
    r = norms.layernorm(same, None, b, stats=True)
    assert torch.equal(r.y, b.expand_as(same)) and (r.mean == 3).all()
    gx, gw, gb = norms.layernorm_backward(x[:4], same, r.mean, r.rstd)
    assert torch.isfinite(gx).all() and not gw.any()


def test_rows_that_are_not_finite_stay_alone():
    for cols in (48, 1001, 4096, 17000):
        x = torch.randn(6, cols, device="cuda")
        x[1, cols // 2], x[3, 0], x[4, cols - 1] = float("nan"), float("inf"), -float("inf")
        y = norms.layernorm(x).y
        assert torch.isnan(y[[1, 3, 4]]).all()
        assert torch.equal(y[[0, 2, 5]], norms.layernorm(torch.where(torch.isfinite(x), x, 0.0)).y[[0, 2, 5]])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 127), (2, 128), (5, 129), (40, 1000), (1, 4096), (300, 520), (2, 17000), (3, 20001)])
def test_blocks_out(rows, cols, dtype):
    """The norm in 8-bit blocks: the blocks of y, but for codes whose value lies next to a tie and scales next to a power of two."""
    x, res, w, b, _, _ = make(rows, cols, dtype, 2)
    r = blocks8.layernorm(x, w, b, residual=res)
    h, u, rstd, y = norm(x, res, w, b)
    assert torch.equal(r.h, norms.layernorm(x, w, b, residual=res).h)
    assert r.blocks.q.shape == x.shape and r.blocks.scale.shape == (rows, -(-cols // 128))
    v = values(r.blocks.q, r.blocks.scale)
    step = r.blocks.scale.double().repeat_interleave(128, 1)[:, :cols]
    close(v, y, 2.0 ** -4, step * 2.0 ** -10 + norm_floor(h, u, rstd, w, cols) + 4 * F32 * b.double().abs())   # half an e4m3 step; half the least subnormal, 2^-10
    q, s = blocks(y.float())
    assert (r.blocks.scale.double() != s).float().mean() < 1e-2 and (v != values(q, s)).float().mean() < 1e-2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_autograd(dtype, residual):
    x, res, w, b, g, gh = make(33, 200, dtype, 3)
    leaves = [t.requires_grad_(True) for t in ((x, w, b, res) if residual else (x, w, b))]
    y, h = tp.layernorm(x, w, b, residual=res if residual else None)
    grads = torch.autograd.grad((y, h), leaves, (g, gh))
    hd, u, rstd, _ = norm(h.detach())
    wx, ww, wb = norm_backward(g, u, rstd, w.detach(), gh)
    size = float((rstd * (1 + u.abs().amax()) ** 2).max()) * float(g.abs().max()) * 2
    off = HALF[dtype] * 2 if residual else 0   # mean and rstd are the unrounded sum's
    close(grads[0], wx, 1.01 * HALF[dtype], (64 * F32 + 4 * off) * size)
    close(grads[1], ww, 1.01 * HALF[dtype], (64 * F32 + 4 * off) * 33 * float(g.abs().max()) * float(u.abs().max()))
    close(grads[2], wb, 1.01 * HALF[dtype], 64 * F32 * 33 * float(g.abs().max()))
    if residual:
        assert torch.equal(grads[0], grads[3])


def test_gradients_against_differences():
    """Central differences of the f64 formula's f32 stand-in: step 2^-6, error of the second order below 1e-3 of the gradients' size."""
    x, res, w, b, g, gh = (t[:4] if t.dim() == 2 else t for t in make(4, 24, torch.float32, 4))
    leaves = [t.requires_grad_(True) for t in (x, res, w, b)]
    y, h = tp.layernorm(x, w, b, residual=res)
    grads = torch.autograd.grad((y, h), leaves, (g, gh))
    with torch.no_grad():
        for leaf, grad in zip(leaves, grads):
            flat, want = leaf.view(-1), torch.empty_like(grad).view(-1)
            for i in range(flat.numel()):
                at, d = float(flat[i]), 2.0 ** -6
                value = []
                for v in (at + d, at - d):
                    flat[i] = v
                    yy, hh = norms.layernorm(x, w, b, residual=res)[:2]
                    value.append(float((yy.double() * g).sum() + (hh.double() * gh).sum()))
                flat[i] = at
                want[i] = (value[0] - value[1]) / (2 * d)
            assert float((grad.view(-1) - want).norm() / want.norm()) < 2e-3


def test_only_what_is_asked_for():
    x, res, w, b, g, _ = make(5, 40, torch.float32)
    assert not tp.layernorm(x, w, b)[0].requires_grad
    w.requires_grad_(True)
    y, h = tp.layernorm(x, w, b)
    assert not h.requires_grad or h.grad_fn is not None
    (gw,) = torch.autograd.grad(y, w, g)
    assert torch.equal(gw, norms.layernorm_backward(g, x, *norms.layernorm(x, w, b, stats=True)[2:], w.detach())[1])
    x.requires_grad_(True)
    y, h = tp.layernorm(x, w, b)
    assert torch.equal(torch.autograd.grad(h, x, g)[0], g)
    y, _ = tp.layernorm(x, w, b)
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=False)   # an expanded gradient
    assert torch.isfinite(gx).all()
    y, _ = tp.layernorm(x, w, b)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_other_streams_and_capture():
    x, res, w, b, g, gh = make(50, 1000, torch.bfloat16)
    want = norms.layernorm(x, w, b, residual=res, stats=True)
    back = norms.layernorm_backward(g, want.h, want.mean, want.rstd, w, gh)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norms.layernorm_backward(g, want.h, want.mean, want.rstd, w, gh)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = norms.layernorm(x, w, b, residual=res, stats=True)
        grads = norms.layernorm_backward(g, r.h, r.mean, r.rstd, w, gh)
    for _ in range(3):
        for t in (*r, *grads):
            t.fill_(7)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip((*r, *grads), (*want, *back)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", [(900, 4097), (900, 4600), (611, 5001), (640, 5120), (450, 5121)])
def test_many_wide_rows(rows, cols, dtype):
    """Around the widths of which an SM works on two rows at once, several rows to each."""
    test_forward(rows, cols, dtype)
    test_blocks_out(rows, cols, dtype)
