"""8-bit rows on the GPU against plain 64-bit implementations.

Tolerances are worst-case bounds of the arithmetic, written where they are
used: U = 2^-24 is f32's unit rounding, OUT[dtype] that of the output type."""
import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import rows8
from tropical_gemm.rows8 import Rows8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
OUT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-37}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# what carrying a factor of a product costs: bf16 rounds the 8-bit operand's
# values once (2^-8 by the unit of bf16's rounding); 16 and 24 bits else
FACTOR = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -15, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def rand8(g, rows, cols):
    return Rows8(torch.randint(-127, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int8),
                 torch.rand(rows, generator=g, device="cuda") * 0.02 + 1e-3)


def values(r):
    return r.q.double() * r.scale.double()[..., None]


def assert_near(got, want, tol):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off - tol).max())} beyond its bound"


def check_rows(r, y, rel):
    """`r` holds y in 8-bit rows; rel: y's own relative error before the
    rounding.  scale = top / 127 within rel + 2U, and each value within half a
    step plus what a relative error makes of 127 steps."""
    top = y.abs().amax(-1)
    assert_near(r.scale, top / 127, top / 127 * (rel + 4 * U) + 2.0 ** -149)
    step = r.scale.double()[..., None]
    assert_near(values(r), y, step * (0.5 + 127 * (2 * rel + 8 * U)))
    assert int(r.q.to(torch.int32).abs().max() if r.q.numel() else 0) <= 127


# ------------------------------------------------------------------ quantize
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 8), (3, 17), (5, 256), (130, 511), (1000, 96), (2, 8192), (7, 32768),
                                        (3, 32776), (2, 100001)])
def test_quantize_and_back(dtype, rows, cols):
    g = gen(rows * cols)
    x = randn(g, rows, cols, dtype=dtype)
    r = rows8.quantize(x)
    check_rows(r, x.double(), 0.0)
    for dt in TYPES:
        assert torch.equal(rows8.dequantize(r, dt), (r.q.float() * r.scale[:, None]).to(dt))


def test_quantize_rounds_half_to_even():
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5, -127.0]], device="cuda")
    assert rows8.quantize(x).q.tolist() == [[127, 0, 2, 2, 0, -2, 64, -127]]


@pytest.mark.parametrize("cols", [8, 9, 40000])
def test_quantize_zero_tiny_and_non_finite_rows(cols):
    x = torch.ones(7, cols, device="cuda")
    x[1] = 0
    x[2] = 1e-38
    x[3, cols // 2] = float("nan")
    x[4, 0] = float("-inf")
    x[5] = 3e38
    x[6] = 1e-30
    r = rows8.quantize(x)
    v = rows8.dequantize(r, torch.float32)
    assert torch.equal(v[1], torch.zeros(cols, device="cuda")) and torch.equal(v[2], torch.zeros(cols, device="cuda"))
    assert torch.isnan(v[3]).all() and torch.isnan(v[4]).all()
    for i in (0, 5, 6):
        assert (r.q[i] == 127).all() and torch.isfinite(r.scale[i])


def test_quantize_strided_and_shaped():
    g = gen(5)
    big = randn(g, 40, 200)
    for view in (big[:, :64], big[::2, 8:72], big[:, 3:70], big.t(), big[::3, ::2], big.reshape(4, 10, 200)[:, :, 5:50],
                 big[:1].expand(6, 200), big[:0], big.reshape(2, 2, 10, 200)):
        r, want = rows8.quantize(view), rows8.quantize(view.contiguous())
        assert r.q.shape == view.shape and torch.equal(r.q, want.q) and torch.equal(r.scale, want.scale)
    assert rows8.quantize(torch.zeros(3, 0, device="cuda")).scale.tolist() == [0, 0, 0]
    sub = Rows8(rows8.quantize(big).q[:, 3:50], rows8.quantize(big).scale)
    assert torch.equal(rows8.dequantize(sub, torch.float32), sub.q.float() * sub.scale[:, None])


# ------------------------------------------------------------------- rmsnorm
NORM_SIZES = [(1, 1), (1, 4096), (3, 17), (33, 256), (300, 511), (700, 1024), (5, 1111), (400, 8192), (2, 32768), (3, 33000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", NORM_SIZES)
@pytest.mark.parametrize("with_residual", [True, False])
def test_rmsnorm(dtype, rows, cols, with_residual):
    g = gen(rows + cols)
    x = randn(g, rows, cols, dtype=dtype)
    res = randn(g, rows, cols, dtype=dtype) * 3 if with_residual else None
    w = randn(g, cols, dtype=dtype)
    n = rows8.rmsnorm(x, w, residual=res, eps=1e-5, checkpoint=True)
    h32 = x.float() + res.float() if with_residual else x.float()
    h = h32.double()
    u = (h.square().mean(-1) + 1e-5).rsqrt()
    # the sum of squares: at most 64 terms in one thread and 64 sums joined, all
    # positive, then root, division and two products; half of it through the root
    rel = (0.5 * 128 + 6) * U
    check_rows(n.rows, h * u[:, None] * w.double(), rel)
    check_rows(n.checkpoint, h, 0.0)
    assert_near(n.rstd, u, u * rel)
    assert torch.equal(n.h, h32.to(dtype))
    plain = rows8.rmsnorm(x, w, residual=res, eps=1e-5)
    assert plain.checkpoint is None and plain.rstd is None
    assert torch.equal(plain.rows.q, n.rows.q) and torch.equal(plain.rows.scale, n.rows.scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols, ld, first", [(700, 13, 13, 0), (900, 1001, 1001, 0), (650, 8185, 8185, 0), (600, 16380, 16380, 0),
                                                   (800, 250, 264, 0), (800, 250, 264, 3), (800, 256, 264, 5), (20, 77, 81, 2), (5, 3, 9, 4)])
def test_rows_that_start_anywhere(dtype, rows, cols, ld, first):
    """Rows off the 16-byte boundaries, all operands alike or not, against the same rows packed."""
    g = gen(rows + cols)

    def view(t):   # the same values at an offset inside a wider matrix
        wide = torch.full((rows, ld), float("nan"), device="cuda", dtype=torch.float32).to(t.dtype)
        wide[:, first:first + cols] = t
        return wide[:, first:first + cols]

    x, res, gr, w = (randn(g, *s, dtype=dtype) for s in ((rows, cols), (rows, cols), (rows, cols), (cols,)))
    x[::7] = 0
    res[::7] = 0
    n = rows8.rmsnorm(x, w, residual=res, checkpoint=True, eps=1e-5)
    h = (x.float() + res.float()).double()
    u = (h.square().mean(-1) + 1e-5).rsqrt()
    check_rows(n.rows, h * u[:, None] * w.double(), (0.5 * 128 + 6) * U)
    check_rows(n.checkpoint, h, 0.0)
    assert torch.equal(n.h, (x.float() + res.float()).to(dtype))
    m = rows8.rmsnorm(view(x), w, residual=view(res), checkpoint=True, eps=1e-5)
    for a, b in ((n.rows, m.rows), (n.checkpoint, m.checkpoint)):
        assert_near(values(a), values(b), 1.001 * a.scale.double()[:, None])   # a step at most: the sums' order may differ
    check_rows(rows8.quantize(view(x)), x.double(), 0.0)
    d = Rows8(n.rows.q, n.rows.scale)
    assert torch.equal(rows8.dequantize(Rows8(view(d.q.float()).to(torch.int8), d.scale), dtype), rows8.dequantize(d, dtype))
    dx, dw = rows8.rmsnorm_backward(gr, n.checkpoint, n.rstd, w, grad_h=res)
    dx2, dw2 = rows8.rmsnorm_backward(view(gr), n.checkpoint, n.rstd, w, grad_h=view(res))
    v, ud = values(n.checkpoint) * n.rstd.double()[:, None], n.rstd.double()[:, None]
    G, W, H = gr.double(), w.double(), res.double()
    want_x, want_w = norm_gradients(G, v, ud[:, 0], W, H)
    c_abs = (G * W * v).abs().mean(-1, keepdim=True)
    tol = 8 * U * (ud * (G * W).abs() + ud * v.abs() * c_abs + H.abs()) + ud * v.abs() * c_abs * 140 * U
    for a, b in ((dx, dw), (dx2, dw2)):
        assert_near(a, want_x, tol + want_x.abs() * OUT[dtype] + TINY[dtype])
        assert_near(b, want_w, (G * v).abs().sum(0) * (rows + 12) * U + want_w.abs() * OUT[dtype] + TINY[dtype])


def test_rmsnorm_of_zero_huge_and_non_finite_rows():
    x = torch.ones(6, 64, device="cuda")
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 9] = float("inf")
    x[4] = 1e15
    x[5] = 1e-15
    w = torch.full((64,), 1e15, device="cuda")
    n = rows8.rmsnorm(x, w, eps=0.0 + 1e-6, checkpoint=True)
    v = rows8.dequantize(n.rows, torch.float32)
    assert torch.equal(v[1], torch.zeros(64, device="cuda"))
    assert torch.isnan(v[2]).all() and torch.isnan(v[3]).all()
    want = x[[0, 4, 5]].double()
    want = want * (want.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * 1e15
    assert_near(v[[0, 4, 5]], want, want * 1e-5)


def test_rmsnorm_shapes_strides_and_streams():
    g = gen(11)
    big, res, w = randn(g, 6, 50, 300), randn(g, 6, 50, 300), randn(g, 300)
    a = rows8.rmsnorm(big[:, ::2, 8:136], w[8:136], residual=res[:, 1::2, 100:228], checkpoint=True)
    b = rows8.rmsnorm(big[:, ::2, 8:136].contiguous(), w[8:136].contiguous(), residual=res[:, 1::2, 100:228].contiguous(), checkpoint=True)
    assert a.rows.q.shape == (6, 25, 128) and a.rows.scale.shape == (6, 25)
    for s, t in ((a.rows.q, b.rows.q), (a.rows.scale, b.rows.scale), (a.h, b.h), (a.checkpoint.q, b.checkpoint.q), (a.rstd, b.rstd)):
        assert torch.equal(s, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = big * 2 - big
        c = rows8.rmsnorm(x, w, residual=res)
        z = rows8.matmul(c.rows, rows8.quantize(big[0]))
    side.synchronize()
    d = rows8.rmsnorm(big, w, residual=res)
    assert torch.equal(c.rows.q, d.rows.q) and torch.equal(z, rows8.matmul(d.rows, rows8.quantize(big[0])))
    e = rows8.rmsnorm(big[:0], w, residual=res[:0], checkpoint=True)
    assert e.rows.q.shape == (0, 50, 300) and e.rstd.shape == (0, 50)


def norm_gradients(grad, v, u, w, gh):
    c = (grad * w * v).mean(-1, keepdim=True)
    return u[:, None] * (grad * w - v * c) + gh, (grad * v).sum(0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("f32_grad", [False, True])
@pytest.mark.parametrize("rows, cols", NORM_SIZES + [(0, 40), (2000, 64), (1, 33001)])
def test_rmsnorm_backward(dtype, f32_grad, rows, cols):
    g = gen(rows * 3 + cols)
    ck = rand8(g, rows, cols)
    u = (values(ck).square().mean(-1) + 1e-6).rsqrt().float()
    w, grad, gh = randn(g, cols, dtype=dtype), randn(g, rows, cols, dtype=torch.float32 if f32_grad else dtype), randn(g, rows, cols, dtype=dtype)
    dx, dw = rows8.rmsnorm_backward(grad, ck, u, w, grad_h=gh)
    v, G, W, H, ud = values(ck) * u.double()[:, None], grad.double(), w.double(), gh.double(), u.double()[:, None]
    want_x, want_w = norm_gradients(G, v, ud[:, 0], W, H)
    c_abs = (G * W * v).abs().mean(-1, keepdim=True)
    # the mean: at most 64 terms per thread and 64 joined, each a few roundings
    tol = 8 * U * (ud * (G * W).abs() + ud * v.abs() * c_abs + H.abs()) + ud * v.abs() * c_abs * 140 * U
    assert dx.dtype == dtype and dw.dtype == dtype
    assert_near(dx, want_x, tol + want_x.abs() * OUT[dtype] + TINY[dtype])
    assert_near(dw, want_w, (G * v).abs().sum(0) * (rows + 12) * U + want_w.abs() * OUT[dtype] + TINY[dtype])
    if rows:
        dx0, dw0 = rows8.rmsnorm_backward(grad, ck, u, w)
        assert_near(dx0, want_x - H, tol + (want_x - H).abs() * OUT[dtype] + TINY[dtype])
        assert torch.equal(dw, dw0)
        again = rows8.rmsnorm_backward(grad, ck, u, w, grad_h=gh)   # a fixed order of the sums
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def lossless(g, rows, cols, scale):
    """Values that 8-bit rows hold exactly: integers with a 127, times a power of two."""
    q = torch.randint(-126, 127, (rows, cols), generator=g, device="cuda").float()
    q[:, cols // 2] = 127
    return q * scale


def test_norm_gradient_against_differences():
    g = gen(3)
    x = lossless(g, 4, 13, 2.0 ** -6)
    w, G, H = randn(g, 13), randn(g, 4, 13), randn(g, 4, 13)
    n = rows8.rmsnorm(x, w, eps=1e-6, checkpoint=True)
    assert torch.equal(rows8.dequantize(n.checkpoint, torch.float32), x)
    dx, dw = rows8.rmsnorm_backward(G, n.checkpoint, n.rstd, w, grad_h=H)

    def loss(xx, ww):
        return (G.double() * xx * (xx.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * ww).sum() + (H.double() * xx).sum()

    X, W, d = x.double(), w.double(), 1e-5
    for i in range(4):
        for j in range(13):
            e = torch.zeros_like(X)
            e[i, j] = d
            diff = float(loss(X + e, W) - loss(X - e, W)) / (2 * d)
            # central differences: d^2 times the third derivative (of order 10 at rows of
            # size 1), and 1e-16 * loss / d; then the kernel's own f32 arithmetic
            assert abs(float(dx[i, j]) - diff) < 1e-5
    for j in range(13):
        e = torch.zeros_like(W)
        e[j] = d
        assert abs(float(dw[j]) - float(loss(X, W + e) - loss(X, W - e)) / (2 * d)) < 1e-5


# -------------------------------------------------------------------- matmul
GEMM_SIZES = [(1, 1, 1), (1, 4096, 4096), (2, 100, 0), (1, 8, 15), (3, 17, 33), (16, 128, 128), (17, 129, 127), (64, 257, 500),
              (65, 1000, 1111), (129, 31, 2048), (128, 128, 16), (256, 256, 256), (257, 640, 1040), (300, 1531, 1111), (512, 2048, 384),
              (1000, 1000, 64), (1025, 513, 4112), (2048, 4096, 512), (2500, 3001, 272), (7, 8200, 16384), (5, 40, 131071)]


def matmul_case(m, n, k, dtype, with_bias, seed=0):
    g = gen(m + n + k + seed)
    a, b = rand8(g, m, k), rand8(g, n, k)
    bias = randn(g, n, dtype=dtype) if with_bias else None
    return a, b, bias


def check_matmul(z, a, b, bias, dtype):
    prod = (a.q.double() @ b.q.double().t()) * a.scale.double()[:, None] * b.scale.double()
    want = prod + (bias.double() if bias is not None else 0)
    # the exact integer sum rounded to f32, two products, the bias' addition
    assert_near(z, want, prod.abs() * 4 * U + want.abs() * (U + OUT[dtype]) + TINY[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", GEMM_SIZES)
def test_matmul(dtype, m, n, k):
    for with_bias in (False, True):
        a, b, bias = matmul_case(m, n, k, dtype, with_bias)
        z = rows8.matmul(a, b, bias=bias, dtype=dtype)
        assert z.dtype == dtype and z.shape == (m, n)
        check_matmul(z, a, b, bias, dtype)


def test_matmul_extreme_sums_are_exact():
    """All products of one sign at the longest sum: 131071 * 127^2 < 2^31."""
    k = 131071
    q = torch.full((2, k), 127, dtype=torch.int8, device="cuda")
    one = torch.ones(2, device="cuda")
    z = rows8.matmul(Rows8(q, one), Rows8(torch.cat([q[:1], -q[:1], q[:1]]), torch.ones(3, device="cuda")), dtype=torch.float32)
    assert z.tolist() == [[float(torch.tensor(v, dtype=torch.float32)) for v in (k * 16129, -k * 16129, k * 16129)]] * 2
    with pytest.raises(rows8.N.TropicalGemmError, match="131072"):
        rows8.matmul(Rows8(torch.zeros(1, 1 << 17, dtype=torch.int8, device="cuda"), one[:1]),
                     Rows8(torch.zeros(1, 1 << 17, dtype=torch.int8, device="cuda"), one[:1]))


@pytest.mark.parametrize("m", [1, 40, 700])
def test_matmul_strides_shapes_and_special_scales(m):
    g = gen(m)
    big_a, big_b = rand8(g, 2 * m, 700), rand8(g, 300, 700)
    for lo, hi in ((0, 640), (16, 528), (3, 600), (100, 101)):
        a = Rows8(big_a.q[::2, lo:hi], big_a.scale[::2])
        b = Rows8(big_b.q[:250, lo:hi], big_b.scale[:250])
        z = rows8.matmul(a, b, dtype=torch.float32)
        check_matmul(z, a, b, None, torch.float32)
    a3 = Rows8(big_a.q.view(2, m, 700), big_a.scale.view(2, m))
    assert torch.equal(rows8.matmul(a3, big_b).view(2 * m, 300), rows8.matmul(big_a, big_b))
    assert rows8.matmul(Rows8(big_a.q[:0], big_a.scale[:0]), big_b).shape == (0, 300)
    assert rows8.matmul(big_a, Rows8(big_b.q[:0], big_b.scale[:0])).shape == (2 * m, 0)
    s = big_a.scale.clone()
    s[0] = float("nan")
    sb = big_b.scale.clone()
    sb[1] = 0
    z = rows8.matmul(Rows8(big_a.q, s), Rows8(big_b.q, sb), dtype=torch.float32)
    assert torch.isnan(z[0]).all() and not torch.isnan(z[1:]).any() and (z[1:, 1] == 0).all()


def test_matmul_many_values_past_32_bits():
    """Offsets beyond 2^31: the last rows of a 2.2 GB operand."""
    m, n, k = 17000, 40, 131000
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    q = torch.zeros(m, k, dtype=torch.int8, device="cuda")
    tail = rand8(gen(1), 300, k)
    q[-300:] = tail.q
    b = rand8(gen(2), n, k)
    z = rows8.matmul(Rows8(q, torch.ones(m, device="cuda")), b, dtype=torch.float32)
    check_matmul(z[-300:], Rows8(tail.q, torch.ones(300, device="cuda")), b, None, torch.float32)
    assert (z[:-300] == 0).all()
    x = rows8.dequantize(Rows8(q, torch.ones(m, device="cuda")), torch.bfloat16)
    assert torch.equal(x[-300:], tail.q.to(torch.bfloat16))
    r = rows8.quantize(x)
    top = tail.q.abs().amax(1).float()
    assert torch.equal(r.scale[-300:], top / 127) and (r.scale[:-300] == 0).all()
    grad = torch.zeros(m, 8, device="cuda", dtype=torch.bfloat16)
    grad[-1, 3] = 2
    _, gb = rows8.matmul_backward(grad, Rows8(q, torch.ones(m, device="cuda")), None)
    assert torch.equal(gb[3], 2 * tail.q[-1].to(torch.bfloat16)) and (gb[:3] == 0).all()


# ----------------------------------------------------------- matmul backward
BACK_SIZES = [(1, 1, 1), (1, 128, 64), (0, 20, 24), (5, 7, 9), (33, 64, 127), (64, 128, 256), (100, 300, 200), (130, 257, 520),
              (512, 512, 256), (777, 1000, 333), (1024, 768, 1280), (2048, 512, 4096), (4096, 1024, 136), (3, 5000, 260), (9000, 40, 48)]


def check_backward(got, g, r, dtype, gdtype):
    """got = g r-values; sums of `n` products in f32 with one rounding (or
    truncation) per step at most."""
    v = values(r)
    want, mag = g.double() @ v, g.double().abs() @ v.abs()
    n = g.shape[1]
    assert_near(got, want, mag * (FACTOR[gdtype] + (n + 8) * 2 * U) + want.abs() * OUT[dtype] + TINY[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", BACK_SIZES)
def test_matmul_backward(dtype, m, n, k):
    g = gen(m * 7 + n + k)
    a, b = rand8(g, m, k), rand8(g, n, k)
    grad = randn(g, m, n, dtype=dtype)
    ga, gb = rows8.matmul_backward(grad, a, b)
    assert ga.dtype == dtype and ga.shape == (m, k) and gb.shape == (n, k)
    check_backward(ga, grad, b, dtype, dtype)
    check_backward(gb, grad.t(), a, dtype, dtype)
    for other in TYPES:
        if other != dtype:
            ga, gb = rows8.matmul_backward(grad, a, b, dtype_a=other, dtype_b=other)
            check_backward(ga, grad, b, other, dtype)
            check_backward(gb, grad.t(), a, other, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_matmul_backward_strides_and_none(dtype):
    g = gen(9)
    big, bigb, grad = rand8(g, 400, 500), rand8(g, 300, 500), randn(g, 400, 310, dtype=dtype)
    for lo, hi in ((0, 480), (16, 416), (5, 333)):
        a, b = Rows8(big.q[:, lo:hi], big.scale), Rows8(bigb.q[:, lo:hi], bigb.scale)
        for gr in (grad[:, :300], grad[:, 7:307]):
            ga, gb = rows8.matmul_backward(gr, a, b)
            check_backward(ga, gr, b, dtype, dtype)
            check_backward(gb, gr.t(), a, dtype, dtype)
    assert rows8.matmul_backward(grad[:, :300], big, None)[0] is None
    assert rows8.matmul_backward(grad[:, :300], None, bigb)[1] is None
    one = torch.ones(1, 1, device="cuda", dtype=dtype).expand(400, 300)   # what sum().backward() hands in
    _, gb = rows8.matmul_backward(one, big, None)
    check_backward(gb, one.t(), big, dtype, dtype)
    grad3 = grad[:, :300].reshape(20, 20, 300)
    a3 = Rows8(big.q.view(20, 20, 500), big.scale.view(20, 20))
    x, y = rows8.matmul_backward(grad3, a3, bigb)
    x2, y2 = rows8.matmul_backward(grad3.reshape(400, 300), big, bigb)
    assert x.shape == (20, 20, 500) and torch.equal(x.view(400, 500), x2) and torch.equal(y, y2)


@pytest.mark.parametrize("dtype", TYPES)
def test_matmul_backward_of_nothing(dtype):
    """Sums of no terms are zero, outputs of no rows or columns are empty."""
    g = gen(1)
    ga, gb = rows8.matmul_backward(randn(g, 5, 0, dtype=dtype), rand8(g, 5, 8), rand8(g, 0, 8))
    assert ga.shape == (5, 8) and not ga.any() and gb.shape == (0, 8)
    ga, gb = rows8.matmul_backward(randn(g, 0, 6, dtype=dtype), rand8(g, 0, 8), rand8(g, 6, 8))
    assert ga.shape == (0, 8) and gb.shape == (6, 8) and not gb.any()
    ga, gb = rows8.matmul_backward(randn(g, 5, 6, dtype=dtype), rand8(g, 5, 0), rand8(g, 6, 0))
    assert ga.shape == (5, 0) and gb.shape == (6, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_matmul_backward_of_a_long_sum(dtype):
    """A sum over two million rows, few outputs and many."""
    g = gen(6)
    r = 2_000_003
    a = Rows8(torch.randint(-127, 128, (r, 24), generator=g, device="cuda", dtype=torch.int8), torch.full((r,), 2.0 ** -9, device="cuda"))
    grad = randn(g, r, 8, dtype=dtype)
    _, gb = rows8.matmul_backward(grad, a, None, dtype_b=torch.float32)
    v = values(a)
    want, mag = grad.double().t() @ v, grad.double().abs().t() @ v.abs()
    # power-of-two scales: the bf16 factors are exact.  Sums of 2e6 terms with a
    # rounding or truncation each 16 terms
    assert_near(gb, want, mag * (2.0 ** -22 + r / 16 * 2 * U))


@pytest.mark.parametrize("dtype", TYPES)
def test_matmul_backward_non_finite(dtype):
    """A NaN gradient reaches what it is a factor of, and nothing else."""
    g = gen(2)
    a, b, grad = rand8(g, 300, 200), rand8(g, 260, 200), randn(g, 300, 260, dtype=dtype)
    grad[7, 9] = float("nan")
    ga, gb = rows8.matmul_backward(grad, a, b)
    assert torch.isnan(ga[7]).all() and torch.isnan(gb[9]).all()
    ga[7], gb[9] = 0, 0
    assert torch.isfinite(ga).all() and torch.isfinite(gb).all()


def test_products_are_bit_stable():
    g = gen(21)
    a, b, grad = rand8(g, 1500, 1000), rand8(g, 900, 1000), randn(g, 1500, 900)
    first = (rows8.matmul(a, b), *rows8.matmul_backward(grad, a, b), *rows8.matmul_backward(grad.bfloat16(), a, b))
    for _ in range(3):
        again = (rows8.matmul(a, b), *rows8.matmul_backward(grad, a, b), *rows8.matmul_backward(grad.bfloat16(), a, b))
        assert all(torch.equal(x, y) for x, y in zip(first, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", [(0, 5), (1, 1), (3, 1000), (1000, 3), (5000, 257), (40000, 16)])
def test_column_sum(dtype, rows, cols):
    x = randn(gen(rows + cols), rows, cols, dtype=dtype)
    for out in (None, torch.float32):
        s = rows8.column_sum(x, out)
        want = x.double().sum(0)
        assert_near(s, want, x.double().abs().sum(0) * (rows + 8) * U + want.abs() * OUT[s.dtype] + TINY[s.dtype])


# ------------------------------------------------------------------ autograd
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", [(5, 7, 9), (200, 136, 264), (64, 256, 512)])
def test_autograd_layer(dtype, m, n, k):
    g = gen(m)
    x, res, nw = randn(g, m, k, dtype=dtype), randn(g, m, k, dtype=dtype), randn(g, k, dtype=dtype)
    w, bias = randn(g, n, k, dtype=dtype) * k ** -0.5, randn(g, n, dtype=dtype)
    leaves = [t.requires_grad_(True) for t in (x, res, nw, w, bias)]
    z, h = tp.rmsnorm_linear_rows8(x, nw, w, residual=res, bias=bias, eps=1e-6)
    gz, gh = randn(g, m, n, dtype=dtype), randn(g, m, k, dtype=dtype)
    gx, gr, gnw, gw, gbias = torch.autograd.grad((z, h), leaves, (gz, gh))
    with torch.no_grad():
        r = rows8.rmsnorm(x, nw, residual=res, eps=1e-6, checkpoint=True)
        b = rows8.quantize(w)
        assert torch.equal(z, rows8.matmul(r.rows, b, bias=bias, dtype=dtype)) and torch.equal(h, r.h)
        check_backward(gw, gz.t(), r.rows, dtype, dtype)
        v, u = values(r.checkpoint) * r.rstd.double()[:, None], r.rstd.double()
        gy, mag = gz.double() @ values(b), gz.double().abs() @ values(b).abs()
        W = nw.double().abs()
        want_x, want_nw = norm_gradients(gy, v, u, nw.double(), gh.double())
        dy = mag * (FACTOR[dtype] + (n + 8) * 2 * U)   # bound of grad_y's error, through the linear map that follows
        tol = u[:, None] * (dy * W + v.abs() * (dy * W * v.abs()).mean(-1, keepdim=True))
        size = u[:, None] * (gy.abs() * W + v.abs() * (gy.abs() * W * v.abs()).mean(-1, keepdim=True)) + gh.double().abs()
        assert_near(gx, want_x, tol + size * 160 * U + want_x.abs() * OUT[dtype] + TINY[dtype])
        assert torch.equal(gx, gr)
        assert_near(gnw, want_nw, (dy * v.abs()).sum(0) + (gy * v).abs().sum(0) * (m + 12) * U + want_nw.abs() * OUT[dtype] + TINY[dtype])
        assert torch.equal(gbias, rows8.column_sum(gz))


def test_autograd_partial_needs_and_frozen_weight():
    g = gen(4)
    x, nw, w = randn(g, 3, 10, 64), randn(g, 64), randn(g, 24, 64)
    frozen = rows8.quantize(w)
    x.requires_grad_(True)
    z, h = tp.rmsnorm_linear_rows8(x, nw, frozen)
    assert z.shape == (3, 10, 24) and h.shape == x.shape and torch.equal(h, x)
    (gx,) = torch.autograd.grad(z.sum(), x, retain_graph=True)
    (gh,) = torch.autograd.grad(h.sum(), x, retain_graph=True)
    (both,) = torch.autograd.grad(z.sum() + h.sum(), x)
    assert torch.equal(gh, torch.ones_like(x))
    assert_near(both, gx.double() + 1, (gx.double().abs() + 1) * 4 * U)
    x = x.detach()
    w.requires_grad_(True)
    z, _ = tp.rmsnorm_linear_rows8(x, nw, w, residual=x)
    (gw,) = torch.autograd.grad(z.sum(), w)
    r = rows8.rmsnorm(x, nw, residual=x)
    check_backward(gw, torch.ones(24, 30, device="cuda"), Rows8(r.rows.q.view(30, 64), r.rows.scale.view(30)), torch.float32, torch.float32)
    with torch.no_grad():
        z2, _ = tp.rmsnorm_linear_rows8(x, nw, w, residual=x)
    assert torch.equal(z, z2) and not z2.requires_grad


def test_autograd_refuses_a_second_derivative():
    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    z, _ = tp.rmsnorm_linear_rows8(x, torch.ones(32, device="cuda"), torch.randn(8, 32, device="cuda"))
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(z.sum(), x, create_graph=True)


def test_linear_gradient_against_differences():
    """z is bilinear in the held values: differences are exact up to rounding."""
    g = gen(8)
    xa, xb = lossless(g, 5, 12, 2.0 ** -5), lossless(g, 6, 12, 2.0 ** -7)
    G = randn(g, 5, 6)
    a, b = rows8.quantize(xa), rows8.quantize(xb)
    assert torch.equal(rows8.dequantize(a, torch.float32), xa) and torch.equal(rows8.dequantize(b, torch.float32), xb)
    ga, gb = rows8.matmul_backward(G, a, b)

    def loss(p, q):
        return float((G.double() * (p @ q.t())).sum())

    A, B, d = xa.double(), xb.double(), 2.0 ** -10
    for i in range(5):
        for j in range(12):
            e = torch.zeros_like(A)
            e[i, j] = d
            assert abs(float(ga[i, j]) - (loss(A + e, B) - loss(A - e, B)) / (2 * d)) < 1e-5
    for i in range(6):
        for j in range(12):
            e = torch.zeros_like(B)
            e[i, j] = d
            assert abs(float(gb[i, j]) - (loss(A, B + e) - loss(A, B - e)) / (2 * d)) < 1e-5


# ------------------------------------------------------------------ refusals
@pytest.mark.parametrize("call", [
    lambda x, r: rows8.rmsnorm(x, torch.ones(7, device="cuda")),
    lambda x, r: rows8.rmsnorm(x, torch.ones(8, device="cuda", dtype=torch.bfloat16)),
    lambda x, r: rows8.rmsnorm(x, torch.ones(8, device="cuda"), residual=x[:2]),
    lambda x, r: rows8.rmsnorm(x, torch.ones(8, device="cuda"), eps=-1.0),
    lambda x, r: rows8.rmsnorm(x, torch.ones(8, device="cuda"), eps=float("nan")),
    lambda x, r: rows8.rmsnorm(x[:, :0], torch.ones(0, device="cuda")),
    lambda x, r: rows8.matmul(r, Rows8(r.q[:, :5], r.scale)),
    lambda x, r: rows8.matmul(r, r, bias=torch.ones(5, device="cuda"), dtype=torch.float32),
    lambda x, r: rows8.matmul(r, r, bias=torch.ones(4, device="cuda"), dtype=torch.bfloat16),
    lambda x, r: rows8.matmul(r, r, dtype=torch.float64),
    lambda x, r: rows8.matmul(r, Rows8(r.q, r.scale.cpu())),
    lambda x, r: rows8.matmul_backward(x, r, None, dtype_b=torch.int32),
    lambda x, r: rows8.matmul_backward(x, Rows8(r.q[:3], r.scale[:3]), None),
    lambda x, r: rows8.matmul_backward(x, None, r),
    lambda x, r: rows8.rmsnorm_backward(x.half(), r, r.scale, torch.ones(8, device="cuda", dtype=torch.bfloat16)),
    lambda x, r: rows8.rmsnorm_backward(x, r, r.scale[:2], torch.ones(8, device="cuda")),
    lambda x, r: rows8.rmsnorm_backward(x[:2], r, r.scale, torch.ones(8, device="cuda")),
    lambda x, r: rows8.rmsnorm_backward(x, r, r.scale, torch.ones(8, device="cuda"), grad_h=x.half()),
])
def test_refusals(call):
    x = torch.ones(4, 8, device="cuda")
    with pytest.raises(ValueError):
        call(x, rows8.quantize(x))


# ------------------------------------------------------------------- example
def test_example_trains_and_serves():
    """The example block learns, and serving gives the trained block's bits:
    the integer sums are exact, whatever kernel a number of tokens takes."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "rows8_block.py")
    spec = importlib.util.spec_from_file_location("rows8_block", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.main(steps=60, tokens=512, width=256)
    assert got["last"] < 0.5 * got["first"]
    assert got["served equals trained"] and got["one token at a time equals all"]


@pytest.mark.parametrize("m", [1, 5, 16, 17, 40, 64, 100, 128, 200, 512, 513, 700])
@pytest.mark.parametrize("n, k", [(16, 16), (130, 1000), (4096, 640), (300, 12000)])
def test_matmul_bits_do_not_depend_on_the_number_of_tokens(m, n, k):
    """Every kernel and split gives the same bits for a token: exact sums, one epilogue."""
    g = gen(n + k)
    a, b = rand8(g, 1024, k), rand8(g, n, k)
    bias = randn(g, n, dtype=torch.bfloat16)
    whole = rows8.matmul(a, b, bias=bias)
    assert torch.equal(rows8.matmul(Rows8(a.q[:m], a.scale[:m]), b, bias=bias), whole[:m])


def test_graph_capture():
    """Norm and product capture into a CUDA graph and replay on new inputs."""
    g = gen(77)
    x, res, w = randn(g, 8, 512, dtype=torch.bfloat16), randn(g, 8, 512, dtype=torch.bfloat16), randn(g, 512, dtype=torch.bfloat16)
    b = rand8(g, 256, 512)

    def run():
        n = rows8.rmsnorm(x, w, residual=res, checkpoint=True)
        z = rows8.matmul(n.rows, b)
        return z, rows8.matmul_backward(z, n.rows, b)[1]

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    x.copy_(randn(g, 8, 512, dtype=torch.bfloat16))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, run()))


def test_products_on_several_streams_at_once():
    """Few-token and paired products, splits and joins, side by side: the same bits as alone."""
    g = gen(31)
    cases = []
    for m, n, k in ((1, 4096, 4096), (40, 1000, 2048), (100, 700, 4096), (700, 1300, 512), (3, 515, 1111)):
        a, b, grad = rand8(g, m, k), rand8(g, n, k), randn(g, m, n)
        cases.append((a, b, grad, grad.bfloat16()))

    def run(c):
        a, b, grad, grad16 = c
        return (rows8.matmul(a, b), *rows8.matmul_backward(grad, a, b), *rows8.matmul_backward(grad16, a, b))

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for turn in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                j = (turn + i) % len(cases)
                got.append((j, run(cases[j])))
    torch.cuda.synchronize()
    for j, r in got:
        assert all(torch.equal(x, y) for x, y in zip(r, want[j]))
