"""Layer norm, 8-bit block linear layers and token log probabilities as they are used together, and what their calls leave alone."""
import importlib.util
import os
import subprocess
import sys

import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import _native as N
from tropical_gemm import blocks8, logprobs, norms
from tropical_gemm.blocks8 import Blocks8
from _layer_forms import HALF, TINY, TYPES, blocks, close, norm, norm_backward, tokens as token_form, values

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODES = {torch.float32: 0, torch.bfloat16: 4, torch.float16: 5}
F32 = 2.0 ** -24
ACC = 2.0 ** -17   # of sum |a||b|: 128 additions of half an f32 step (tensor core), and as many blocks' at most


def held(t, tall=1):
    q, s = blocks(t.detach(), tall)
    return q * s.repeat_interleave(tall, 0)[:t.shape[0]].repeat_interleave(128, 1)[:, :t.shape[1]]


@pytest.mark.parametrize("rows, width, vocab", [(1, 256, 1000), (37, 200, 513), (300, 640, 5000)])
def test_a_step_from_hidden_states_to_gradients(rows, width, vocab):
    """norm -> linear -> log probabilities and back, in f32; each stage against its formula on the stage's own inputs."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    x, r, w, b, weight = (t.requires_grad_(True) for t in (n(rows, width), n(rows, width), 1 + 0.1 * n(width), 0.1 * n(width), n(vocab, width) * width ** -0.5))
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    y, h = tp.layernorm(x, w, b, residual=r)
    z = tp.linear_blocks8(y, weight)
    lp, entropy = tp.token_logprobs(z, ids)
    loss = -lp.mean() - 0.1 * entropy.mean() + 0.01 * h.mean()
    gx, gr, gw, gb, gweight, gz, gy = torch.autograd.grad(loss, (x, r, w, b, weight, z, y))
    wl, we, logs = token_form(z.detach(), ids)
    close(lp, wl, 2 * F32, 2.0 ** -18 + 4 * F32 * float(z.detach().abs().max()))
    p = logs.exp()
    want = (p / rows) + 0.1 / rows * p * (logs + we[:, None])
    want[torch.arange(rows), ids] -= 1 / rows
    close(gz, want, 2 * F32, (2.0 ** -16 / rows) * (p + 1e-3))
    for got, a, c in ((gy, held(gz), held(weight, 128)), (gweight, held(gz.t()), held(y.t()).t())):
        close(got, a @ c, 1.01 * F32, ACC * (a.abs() @ c.abs()) + 2.0 ** -126)
    hd, u, rstd, yd = norm(x.detach(), r.detach(), w.detach(), b.detach())
    wx, ww, wb = norm_backward(gy, u, rstd, w.detach(), torch.full_like(x, 0.01 / (rows * width)))
    size = float(gy.abs().max()) * float((rstd * (1 + u.abs().amax()) ** 2).max()) * 2
    close(gx, wx, F32, 64 * F32 * size)
    assert torch.equal(gx, gr)
    close(gw, ww, F32, 64 * F32 * rows * float(gy.abs().max()) * float(u.abs().max()))
    close(gb, wb, F32, 64 * F32 * rows * float(gy.abs().max()))


def test_serving_equals_its_parts():
    x, r = torch.randn(20, 384, device="cuda").bfloat16(), torch.randn(20, 384, device="cuda").bfloat16()
    w, b, weight = torch.randn(384, device="cuda").bfloat16(), torch.randn(384, device="cuda").bfloat16(), torch.randn(900, 384, device="cuda").bfloat16()
    w8 = blocks8.quantize_tiles(weight)
    n = blocks8.layernorm(x, w, b, residual=r)
    z = blocks8.matmul(n.blocks, w8, dtype=torch.float32)
    v, wv = values(n.blocks.q, n.blocks.scale), values(w8.q, w8.scale)
    close(z, v @ wv.t(), F32, ACC * (v.abs() @ wv.abs().t()))
    a = logprobs.token_logprobs(z, top=4)
    assert torch.equal(a.top_tokens[:, 0], z.argmax(1))
    one = torch.cat([logprobs.token_logprobs(blocks8.matmul(blocks8.layernorm(x[i:i + 1], w, b, residual=r[i:i + 1]).blocks, w8, dtype=torch.float32), top=4).top_tokens
                     for i in range(20)])
    assert (one[:, 0] == a.top_tokens[:, 0]).float().mean() > 0.8   # a code next to a tie may move a near draw


@pytest.mark.parametrize("m, n, k", [(2048, 2048, 1024), (2300, 2100, 1111), (20000, 100, 700), (600, 600, 16384), (768, 768, 40000), (200, 4516, 8594), (351, 122, 20000),
                                     (1024, 4096, 130), (4000, 1300, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_large_products(m, n, k, dtype):
    """Shapes of the paired kernel, whole sums and split ones; scales that are powers of two and others, per row and per tile, and a NaN."""
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, w = torch.randn(m, k, generator=g, device="cuda"), torch.randn(n, k, generator=g, device="cuda") * k ** -0.5
    bias = torch.randn(n, generator=g, device="cuda").to(dtype)
    a = blocks8.quantize(x)
    for b in (blocks8.quantize_tiles(w), blocks8.quantize(w)):
        av, bv = values(a.q, a.scale), values(b.q, b.scale)
        want, size = av @ bv.t(), av.abs() @ bv.abs().t()
        z = blocks8.matmul(a, b, bias=bias, dtype=dtype)
        close(z, want + bias.double(), 1.01 * HALF[dtype], ACC * (size + 1) + TINY[dtype])
        assert torch.equal(z, blocks8.matmul(a, b, bias=bias, dtype=dtype))
        other = Blocks8(a.q, a.scale * 1.25)
        z = blocks8.matmul(other, b, dtype=dtype)
        close(z, 1.25 * want, 1.01 * HALF[dtype], 1.25 * ACC * size + TINY[dtype])
        some = a.scale.clone()
        some[m // 2, 0] = float("nan")
        z = blocks8.matmul(Blocks8(a.q, some), b, dtype=dtype)
        assert torch.isnan(z[m // 2]).all() and torch.isfinite(z).sum() == (m - 1) * n
        some[m // 3, -1] *= 1.5   # one scale among all
        z = blocks8.matmul(Blocks8(a.q, some), b, dtype=dtype)
        assert torch.isnan(z[m // 2]).all()
        rows = torch.arange(m, device="cuda") != m // 2
        some[m // 2, 0] = 0
        av = values(a.q, some)
        close(z[rows], (av @ bv.t())[rows], 1.01 * HALF[dtype], 1.5 * ACC * size[rows] + TINY[dtype])


def test_long_sums_of_one_sign():
    """65,000 terms: what the tensor core may sum by itself is a chunk of 64 blocks, 16 for f32 (an error of 1e-6 at most of sums of one sign)."""
    x, w = torch.rand(700, 65000, device="cuda"), torch.rand(600, 65000, device="cuda")
    a, b = blocks8.quantize(x), blocks8.quantize_tiles(w)
    want = values(a.q, a.scale) @ values(b.q, b.scale).t()
    close(blocks8.matmul(a, b, dtype=torch.float32), want, 2e-6)
    close(blocks8.matmul(a, b), want, HALF[torch.bfloat16] + 8e-6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols", [(1, 40), (5, 129), (700, 200), (900, 1000), (3, 17001)])
def test_outputs_stay_within_their_rows(rows, cols, dtype):
    """Through the C entries, each output with a pitch of its own: what lies between its rows and behind the last one is left as it was."""
    L, e, code = N.lib(), torch.tensor([], dtype=dtype).element_size(), CODES[dtype]
    s = torch.cuda.current_stream().cuda_stream
    x, r, g = (torch.randn(rows, cols, device="cuda").to(dtype) for _ in range(3))
    w, b = torch.randn(cols, device="cuda").to(dtype), torch.randn(cols, device="cuda").to(dtype)

    def out(n, k, pad, dt):
        t = torch.full((n * (k + pad) + 64,), 77, device="cuda", dtype=dt)
        return t, k + pad

    def check(t, n, k, ld):
        left = t.clone()
        body = left[:n * ld].view(n, ld)
        body[:, :k] = 77
        assert (left == 77).all()
        return t[:n * ld].view(n, ld)[:, :k]

    ref = norms.layernorm(x, w, b, residual=r, stats=True)
    for pad_y, pad_h in ((3, 5), (8, 16), (1, 1), (0, 0)):
        (y, ly), (h, lh) = out(rows, cols, pad_y, dtype), out(rows, cols, pad_h, dtype)
        N.check(L.tg_layernorm(code, rows, cols, x.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), b.data_ptr(), 1e-5, h.data_ptr(), lh, y.data_ptr(), ly, None, None, s))
        assert torch.equal(check(h, rows, cols, lh), ref.h)
        close(check(y, rows, cols, ly), ref.y.double(), 4 * HALF[dtype], 64 * F32 * 8)
        (gx, lx) = out(rows, cols, pad_y, dtype)
        gw, gb = torch.full((2, cols + 32), 77, device="cuda", dtype=dtype)
        N.check(L.tg_layernorm_backward(code, rows, cols, g.data_ptr(), cols, None, 0, w.data_ptr(), ref.h.data_ptr(), cols, ref.mean.data_ptr(), ref.rstd.data_ptr(),
                                        gx.data_ptr(), lx, gw.data_ptr(), gb.data_ptr(), s))
        want = norms.layernorm_backward(g, ref.h, ref.mean, ref.rstd, w)
        close(check(gx, rows, cols, lx), want[0].double(), 4 * HALF[dtype], 256 * F32 * float(want[0].abs().max()) + TINY[dtype])
        assert (gw[cols:] == 77).all() and (gb[cols:] == 77).all()
    q, qt = blocks8.quantize_both(x)
    kb, rb = -(-cols // 128), -(-rows // 128)
    for pad in (0, 3, 16):
        (c, lc), (ct, lt) = out(rows, cols, pad, torch.uint8), out(cols, rows, pad, torch.uint8)
        (sc, ls), (st, lst) = out(rows, kb, 1, torch.float32), out(cols, rb, 2, torch.float32)
        total = torch.full((cols + 32,), 77, device="cuda", dtype=dtype)
        N.check(L.tg_blocks8_quantize(code, rows, cols, x.data_ptr(), cols, c.data_ptr(), lc, sc.data_ptr(), ls, 1, ct.data_ptr(), lt, st.data_ptr(), lst, 1, total.data_ptr(), s))
        assert torch.equal(check(c, rows, cols, lc), q.q.view(torch.uint8)) and torch.equal(check(ct, cols, rows, lt), qt.q.view(torch.uint8))
        assert torch.equal(check(sc, rows, kb, ls), q.scale) and torch.equal(check(st, cols, rb, lst), qt.scale)
        close(total[:cols], x.double().sum(0), 1.01 * HALF[dtype], 64 * F32 * x.double().abs().sum(0) + TINY[dtype])
        assert (total[cols:] == 77).all()
        (v, lv) = out(rows, cols, pad, dtype)
        N.check(L.tg_blocks8_dequantize(code, rows, cols, 1, c.data_ptr(), lc, sc.data_ptr(), ls, 1, v.data_ptr(), lv, s))
        assert torch.equal(check(v, rows, cols, lv), blocks8.dequantize(q, dtype))
        wt = blocks8.quantize_tiles(torch.randn(70, cols, device="cuda"))
        (z, lz) = out(rows, 70, pad + 1, dtype)
        N.check(L.tg_blocks8_gemm(code, rows, 70, cols, c.data_ptr(), lc, sc.data_ptr(), ls, 1, wt.q.data_ptr(), wt.q.stride(0), 128, wt.scale.data_ptr(), kb, 1, None, z.data_ptr(), lz, s))
        assert torch.equal(check(z, rows, 70, lz), blocks8.matmul(q, wt, dtype=dtype))
    ids = torch.randint(0, cols, (rows,), device="cuda")
    a = logprobs.token_logprobs(x, ids)
    one = torch.ones(rows, device="cuda")
    want = logprobs.token_logprobs_backward(x, ids, a.stats, a.entropy, one, one)
    for pad in (0, 3, 8):
        (gl, lg) = out(rows, cols, pad, dtype)
        N.check(L.tg_token_logprobs_backward(code, rows, cols, x.data_ptr(), cols, ids.data_ptr(), -100, a.stats.data_ptr(), a.entropy.data_ptr(), one.data_ptr(), one.data_ptr(),
                                             gl.data_ptr(), lg, s))
        assert torch.equal(check(gl, rows, cols, lg), want)
    here = x.clone()   # in place
    N.check(L.tg_token_logprobs_backward(code, rows, cols, here.data_ptr(), cols, ids.data_ptr(), -100, a.stats.data_ptr(), a.entropy.data_ptr(), one.data_ptr(), one.data_ptr(),
                                         here.data_ptr(), cols, s))
    assert torch.equal(here, want)


def test_calls_at_once_on_two_streams():
    x, w, weight = torch.randn(400, 640, device="cuda").bfloat16(), torch.randn(640, device="cuda").bfloat16(), torch.randn(3000, 640, device="cuda").bfloat16()
    g = torch.randn(400, 640, device="cuda").bfloat16()
    w8, ids = blocks8.quantize_tiles(weight), torch.randint(0, 3000, (400,), device="cuda")

    def run():
        s = norms.layernorm(x, w, stats=True)
        b = blocks8.layernorm(x, w)
        z = blocks8.matmul(b.blocks, w8, dtype=torch.float32)
        t = logprobs.token_logprobs(z, ids, top=6)
        return [s.y, *norms.layernorm_backward(g, x, s.mean, s.rstd, w), z, t.logprob, t.entropy, t.top_tokens, *(t.float() for t in blocks8.quantize_both(x)[1])]

    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_two_graphs_replayed_at_once():
    """Captured calls take their scratch into the graph; two graphs on two streams do not share it."""
    x, weight, g = (torch.randn(*s, device="cuda").bfloat16() for s in ((2048, 1024), (2048, 1024), (2048, 2048)))
    x.requires_grad_(True), weight.requires_grad_(True)

    def step():
        z = tp.linear_blocks8(x, weight)
        return [z.detach(), *torch.autograd.grad(z, (x, weight), g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    side.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(p, q) for p, q in zip(out, want))


CAPTURE = """
import sys
sys.path.insert(0, {pkg!r})
import torch
import tropical_gemm.pytorch as tp
x, w, b, v = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((30, 256), (256,), (256,), (400, 256)))
ids = torch.randint(0, 400, (30,), device="cuda")

def step():
    y, h = tp.layernorm(x, w, b)
    return sum(t.sum() for t in tp.token_logprobs(tp.linear_blocks8(y, v), ids)) + h.sum()

side = torch.cuda.Stream()
with torch.cuda.stream(side):
    want = torch.autograd.grad(step(), (x, w, b, v))
torch.cuda.synchronize()
alive = step()
for call in (lambda: tp.layernorm(x, w, b), lambda: tp.linear_blocks8(x, torch.ones(9, 256, device="cuda"), None), lambda: tp.token_logprobs(x, ids % 256)):
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()
    except RuntimeError as e:
        assert "another stream" in str(e), e
    else:
        raise AssertionError("captured")
alive.backward()
assert all(torch.equal(p.grad, q) for p, q in zip((x, w, b, v), want))
del alive
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = torch.autograd.grad(step(), (x, w, b, v))
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(got, want))
print("same")
"""


def test_a_capture_while_an_eager_graph_of_the_leaves_lives_is_refused():
    """Its backward would break the capture off; without that graph it is captured.  In a process of its own."""
    r = subprocess.run([sys.executable, "-c", CAPTURE.format(pkg=os.path.join(ROOT, "tropical-gemm_b200"))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_calls_record_no_graph():
    x, w = torch.randn(6, 256, device="cuda", requires_grad=True), torch.randn(256, device="cuda", requires_grad=True)
    ids = torch.zeros(6, dtype=torch.int64, device="cuda")
    s = norms.layernorm(x, w, w, residual=x, stats=True)
    b = blocks8.layernorm(x, w, w, residual=x)
    t = logprobs.token_logprobs(x, ids, top=2)
    z = blocks8.matmul(b.blocks, blocks8.quantize(x), dtype=torch.float32)
    for o in (*s, b.h, b.blocks.scale, *t, z, *norms.layernorm_backward(x, x, s.mean, s.rstd, w, x), blocks8.dequantize(blocks8.quantize_tiles(x)),
              logprobs.token_logprobs_backward(x, ids, t.stats, t.entropy, s.mean, s.rstd)):
        assert not o.requires_grad and o.grad_fn is None


def test_the_example():
    spec = importlib.util.spec_from_file_location("answer_head", os.path.join(ROOT, "examples", "answer_head.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    r = m.main(steps=5, rows=64, width=128, vocab=300)
    assert all(torch.isfinite(torch.tensor(v)) for v in r.values())
    torch.manual_seed(1)
    head = m.Head(64, 200).cuda()
    x = torch.randn(10, 64, device="cuda")
    lp, h = tp.token_logprobs(head(x), torch.arange(10, device="cuda"))
    (lp.sum() + h.sum()).backward()
    assert all(torch.isfinite(p.grad).all() and p.grad.any() for p in head.parameters())


def test_products_behind_one_another_on_streams():
    """Short sums of many tiles (several thread blocks per SM), clusters and pairs, each kernel started while the one before it ends."""
    products = []
    for m, n, k in [(64, 65536, 128), (17, 30000, 256), (300, 1000, 130), (1, 4096, 4096), (2048, 2048, 512), (64, 20000, 128)]:
        a = blocks8.quantize(torch.randn(m, k, device="cuda").bfloat16())
        b = blocks8.quantize_tiles(torch.randn(n, k, device="cuda").bfloat16())
        products.append((a, b, blocks8.matmul(a, b)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got += [(blocks8.matmul(a, b), z) for a, b, z in products]
    torch.cuda.synchronize()
    assert all(torch.equal(x, z) for x, z in got)


def test_the_same_tensor_twice():
    """x as its own residual: both of its gradients add up."""
    x = torch.randn(300, 4700, device="cuda", requires_grad=True)
    w = torch.randn(4700, device="cuda", requires_grad=True)
    y, h = tp.layernorm(x, w, None, residual=x)
    g = torch.randn_like(y)
    gx, gw = torch.autograd.grad((y, h), (x, w), (g, g))
    xd, wd = (t.detach().double().requires_grad_(True) for t in (x, w))
    hd = 2 * xd
    ex, ew = torch.autograd.grad((torch.nn.functional.layer_norm(hd, (4700,), wd, None, 1e-5), hd), (xd, wd), (g.double(), g.double()))
    # f32 sums in trees of some 32 steps: 32 half steps of 2^-24, relative to the whole
    assert (gx.double() - ex).norm() <= 32 * 2.0 ** -24 * ex.norm() and (gw.double() - ew).norm() <= 32 * 2.0 ** -24 * ew.norm()
