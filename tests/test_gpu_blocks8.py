"""8-bit floating point blocks on the GPU: quantisation bit by bit, products and their gradients against 64 bits.

A product's tolerance: the tensor core's f32 sums over a block of 128 and the f32 sums of the blocks, as 2^-18 of
sum |a||b| (a 128-term sum may lose 128 half steps of f32, 2^-17, where every addition rounds the same way; the blocks' sums
a half step each), and one rounding to the output's type."""
import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import blocks8
from tropical_gemm.blocks8 import Blocks8
from _layer_forms import HALF, TINY, TYPES, blocks, close, values

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
ACC = 2.0 ** -17


def hidden(rows, cols, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 104729 + rows * 1009 + cols)
    x = torch.randn(rows, cols, generator=g, device="cuda") * 10 ** (6 * torch.rand(rows, 1, generator=g, device="cuda") - 3)
    return x.to(dtype)


def same(b, x, tall=1):
    q, s = blocks(x, tall)
    assert b.q.dtype == torch.float8_e4m3fn and b.q.shape == x.shape
    assert torch.equal(b.scale.double(), s)
    assert torch.equal(b.q.double(), q)


SIZES = [(1, 1), (1, 128), (2, 7), (3, 129), (128, 128), (127, 255), (130, 1000), (300, 64), (17, 4096), (1000, 513), (256, 16), (513, 1024)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", SIZES)
def test_quantize(rows, cols, dtype):
    x = hidden(rows, cols, dtype)
    same(blocks8.quantize(x), x)
    a, at = blocks8.quantize_both(x)
    same(a, x)
    same(at, x.t().contiguous())
    w = blocks8.quantize_tiles(x)
    same(w, x, 128)
    wt = blocks8.transpose(w)
    assert torch.equal(wt.q.double(), w.q.double().t()) and torch.equal(wt.scale, w.scale.t())
    for b in (a, w):
        close(blocks8.dequantize(b, dtype), values(b.q, b.scale), HALF[dtype] if dtype != torch.float32 else 0.0, TINY[dtype])
        assert b.q.stride(0) % 16 == 0 or rows == 1


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strided(dtype):
    wide = hidden(70, 400, dtype)
    for skip in (1, 2, 3, 4, 8):
        x = wide[:, skip:skip + 301]
        same(blocks8.quantize(x), x)
        a, at = blocks8.quantize_both(x)
        same(a, x)
        same(at, x.t().contiguous())
        same(blocks8.quantize_tiles(x), x, 128)
    x = wide.view(7, 10, 400)[:, 2:9, 5:200]
    b = blocks8.quantize(x)
    assert b.q.shape == x.shape and b.scale.shape == (7, 7, 2)
    same(Blocks8(b.q.reshape(49, 195), b.scale.reshape(49, 2)), x.reshape(49, 195))
    a, at = blocks8.quantize_both(x)
    assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and at.q.shape == (195, 49)
    same(at, x.reshape(49, 195).t())
    t = wide.t()   # elements of a row are not contiguous
    same(blocks8.quantize(t), t)


def test_quantize_ties_and_ends():
    """Every tie of e4m3, subnormals among them; the largest value at and around 448 times a power of two; the least scale."""
    codes = torch.arange(0, 127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    ties = (codes[:-1].double() + codes[1:].double()) / 2
    for sign in (1.0, -1.0):
        x = torch.full((len(ties), 128), 448.0, device="cuda")
        x[:, 1:] = (ties * sign).float()[:, None]
        same(blocks8.quantize(x), x)
    near = torch.tensor([448.0, 448.0 * (1 + 2.0 ** -23), 447.9999, 256.0, 255.99998, 224.0, 1.0, 1.75, 1.7500001], device="cuda")
    for e in (-140, -130, -126, -110, -20, 0, 30, 110, 119):
        x = torch.zeros(len(near), 130, device="cuda")
        x[:, 5] = (near.double() * 2.0 ** e).float()
        x[:, 9] = -x[:, 5] / 3
        x[:, 129] = x[:, 5]
        same(blocks8.quantize(x), x)
        same(blocks8.quantize_tiles(x), x, 128)
    zero = blocks8.quantize(torch.zeros(3, 200, device="cuda"))
    assert (zero.scale == 2.0 ** -126).all() and not zero.q.float().any()
    big = torch.full((2, 128), 3.4028234e38, device="cuda")
    same(blocks8.quantize(big), big)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_quantize_not_finite(bad):
    x = torch.randn(200, 300, device="cuda")
    x[3, 130], x[150, 299] = bad, bad
    for b, turned in ((blocks8.quantize(x), False), (blocks8.quantize_both(x)[0], False), (blocks8.quantize_both(x)[1], True)):
        want = torch.zeros_like(b.scale, dtype=torch.bool)
        if turned:
            want[130, 0] = want[299, 1] = True
        else:
            want[3, 1] = want[150, 2] = True
        assert torch.equal(torch.isnan(b.scale), want)
        v = blocks8.dequantize(b, torch.float32)
        assert torch.equal(torch.isnan(v), want.repeat_interleave(128, 1)[:, :v.shape[1]])
    assert torch.isnan(blocks8.quantize_tiles(x).scale).sum() == 2
    z = blocks8.matmul(blocks8.quantize(x), blocks8.quantize_tiles(torch.randn(40, 300, device="cuda")), dtype=torch.float32)
    assert torch.isnan(z[[3, 150]]).all() and torch.isfinite(z).sum() == 198 * 40


def test_empty():
    e = blocks8.quantize(torch.empty(0, 40, device="cuda"))
    assert e.q.shape == (0, 40) and e.scale.shape == (0, 1)
    w = blocks8.quantize_tiles(torch.randn(9, 40, device="cuda"))
    assert blocks8.matmul(e, w).shape == (0, 9)
    none = blocks8.quantize(torch.empty(5, 0, device="cuda"))
    assert none.scale.shape == (5, 0)
    b = torch.randn(9, device="cuda")
    z = blocks8.matmul(none, blocks8.quantize_tiles(torch.empty(9, 0, device="cuda")), bias=b, dtype=torch.float32)
    assert torch.equal(z, b.expand(5, 9))
    assert blocks8.matmul(blocks8.quantize(torch.randn(5, 40, device="cuda")), blocks8.quantize_tiles(torch.empty(0, 40, device="cuda"))).shape == (5, 0)
    a, at = blocks8.quantize_both(torch.empty(0, 40, device="cuda"))
    assert at.q.shape == (40, 0) and at.scale.shape == (40, 0)


def check_product(a, b, dtype, bias=None):
    z = blocks8.matmul(a, b, bias=bias, dtype=dtype)
    av, bv = values(a.q, a.scale), values(b.q, b.scale)
    want, size = av @ bv.t(), av.abs() @ bv.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    close(z, want, 1.01 * HALF[dtype], ACC * size + TINY[dtype])
    return z


PRODUCTS = [(1, 1, 1), (1, 4096, 4096), (2, 130, 257), (7, 100, 128), (16, 512, 1024), (17, 300, 1000), (33, 64, 5000), (64, 2048, 640), (65, 200, 96), (128, 128, 128),
            (129, 257, 384), (256, 256, 256), (300, 700, 1111), (333, 1531, 520), (513, 1000, 130), (1024, 1024, 2048), (2000, 520, 64), (100, 4000, 3000), (700, 64, 9000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", PRODUCTS)
def test_matmul(m, n, k, dtype):
    x, w = hidden(m, k, torch.float32, 1), hidden(n, k, torch.float32, 2) * k ** -0.5
    if dtype == torch.float16:   # within its range
        x, w = x / x.abs().amax(1, keepdim=True), w / w.abs().amax(1, keepdim=True)
    bias = torch.randn(n, device="cuda").to(dtype)
    a = blocks8.quantize(x)
    for b in (blocks8.quantize_tiles(w), blocks8.quantize(w)):
        z = check_product(a, b, dtype, bias)
        check_product(a, b, dtype)
        assert torch.equal(z, blocks8.matmul(a, b, bias=bias, dtype=dtype))


@pytest.mark.parametrize("m, n, k", [(3, 200, 300), (40, 130, 1000), (300, 300, 700), (70, 5, 129)])
def test_matmul_any_operands(m, n, k):
    """Codes and scales as they come: any pitch and offset, scales with any strides and of any size, transposed weights."""
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    kb = -(-k // 128)
    code = lambda *s: torch.randint(0, 127, s, generator=g, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)   # noqa: E731
    scale = lambda *s: torch.rand(*s, generator=g, device="cuda") * 3   # noqa: E731
    aq, bq = code(m, k + 9)[:, 3:3 + k], code(n, k + 2)[:, 1:1 + k]
    for a_scale in (scale(m, kb), scale(kb, m).t(), scale(m, kb + 3)[:, 1:1 + kb], scale(1, kb).expand(m, kb)):
        for b_scale in (scale(-(-n // 128), kb), scale(kb, -(-n // 128)).t(), scale(n, kb), scale(kb, n).t(), scale(1, 1).expand(n, kb)):
            check_product(Blocks8(aq, a_scale), Blocks8(bq, b_scale), torch.float32)
    a = Blocks8(aq.reshape(1, m, 1, k), scale(m, kb).view(1, m, 1, kb))
    assert blocks8.matmul(a, Blocks8(bq, scale(n, kb))).shape == (1, m, 1, n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (5, 70, 130), (300, 200, 257), (128, 128, 128), (17, 513, 1000), (400, 1000, 300), (1000, 64, 640)])
def test_linear_gradients(m, n, k, dtype):
    """z, grad_x and grad_w are products of quantised operands: exact up to the sums; the bias's gradient is a plain sum."""
    x, w, g = hidden(m, k, torch.float32, 3), hidden(n, k, torch.float32, 4), hidden(m, n, torch.float32, 5)
    x, w, g = (t / t.abs().amax(1, keepdim=True) for t in (x, w, g)) if dtype == torch.float16 else (x, w, g)
    x, w, g, b = (t.to(dtype) for t in (x, w, g, torch.randn(n, device="cuda")))
    for t in (x, w, b):
        t.requires_grad_(True)
    z = tp.linear_blocks8(x, w, b)
    gx, gw, gb = torch.autograd.grad(z, (x, w, b), g)
    held = lambda t, tall=1: (lambda q, s: q * s.repeat_interleave(tall, 0)[:t.shape[0]].repeat_interleave(128, 1)[:, :t.shape[1]])(*blocks(t.detach(), tall))   # noqa: E731
    xv, wv, gv, xt, gt = held(x), held(w, 128), held(g), held(x.t()), held(g.t())
    db = b.detach().double()
    for got, p, q, more in ((z, xv, wv.t(), db), (gx, gv, wv, None), (gw, gt, xt.t(), None)):
        want, size = p @ q, p.abs() @ q.abs()
        if more is not None:
            want, size = want + more, size + more.abs()
        close(got, want, 1.01 * HALF[dtype], ACC * size + TINY[dtype])
    close(gb, g.double().sum(0), 1.01 * HALF[dtype], 2048 * F32 * g.double().abs().sum(0) + TINY[dtype])


def test_linear_gradient_against_the_formula():
    """Beside the unquantised layer: each factor is off by at most half an e4m3 step of 2^-4, or of its block's least steps."""
    x, w, g = (torch.randn(*s, device="cuda") for s in ((200, 300), (150, 300), (200, 150)))
    x.requires_grad_(True), w.requires_grad_(True)
    z = tp.linear_blocks8(x, w)
    gx, gw = torch.autograd.grad(z, (x, w), g)
    xd, wd, gd = x.detach().double(), w.detach().double(), g.double()
    for got, p, q in ((z, xd, wd.t()), (gx, gd, wd), (gw, gd.t(), xd)):
        floor = 2.0 ** -10 * 2.0 ** -6   # subnormal codes: half of 2^-9 of a scale; the scale is below 2^-6 for values below 7
        a, b = p.abs(), q.abs()
        limit = ((a * (1 + 2.0 ** -4) + floor) @ (b * (1 + 2.0 ** -4) + floor)) - a @ b
        assert ((got.detach().double() - p @ q).abs() <= limit).all()
        assert float((got.detach().double() - p @ q).norm() / (p @ q).norm()) < 2 * 2.0 ** -4


def test_linear_frozen_and_needs():
    x, w, b = torch.randn(3, 20, 200, device="cuda", dtype=torch.bfloat16), torch.randn(140, 200, device="cuda", dtype=torch.bfloat16), None
    w8 = blocks8.quantize_tiles(w)
    assert torch.equal(tp.linear_blocks8(x, w8), tp.linear_blocks8(x, w)) and not tp.linear_blocks8(x, w).requires_grad
    x.requires_grad_(True)
    (g1,) = torch.autograd.grad(tp.linear_blocks8(x, w8).sum(), x)
    (g2,) = torch.autograd.grad(tp.linear_blocks8(x, w).sum(), x)
    assert torch.equal(g1, g2) and g1.shape == x.shape
    frozen = Blocks8(w8.q, w8.scale.clone().requires_grad_(True))
    z = tp.linear_blocks8(x.detach(), frozen)
    assert not z.requires_grad
    tp.linear_blocks8(x, frozen).sum().backward()
    assert frozen.scale.grad is None
    with pytest.raises(ValueError, match="tiles"):
        tp.linear_blocks8(x, blocks8.quantize(w))
    assert tp.linear_blocks8(x.detach(), blocks8.quantize(w)).shape == (3, 20, 140)
    w.requires_grad_(True)
    z = tp.linear_blocks8(x.detach(), w)
    (gw,) = torch.autograd.grad(z, w, torch.ones_like(z))
    assert gw.shape == w.shape
    none = tp.linear_blocks8(torch.empty(0, 200, device="cuda", dtype=torch.bfloat16), w)
    assert not torch.autograd.grad(none.sum(), w)[0].any()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(tp.linear_blocks8(x, w).sum(), x, create_graph=True)


def test_linear_other_streams_and_capture():
    x, w, b, g = (torch.randn(*s, device="cuda", dtype=torch.bfloat16) for s in ((80, 300), (200, 300), (200,), (80, 200)))
    for t in (x, w, b):
        t.requires_grad_(True)

    def step():
        z = tp.linear_blocks8(x, w, b)
        return [z.detach(), *torch.autograd.grad(z, (x, w, b), g)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for t in out:
            t.fill_(7)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
