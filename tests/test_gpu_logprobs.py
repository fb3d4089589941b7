"""Token log probabilities on the GPU against 64 bits.

f32 arithmetic: x - m is one rounding (half a step of the largest |x|), the exponential within 2^-21 of itself, sums of up to
2^17 terms in chains of at most 2^9 additions and a tree: log S within 2^-13 at worst, in practice 2^-20; the tests
hold logprob to 2^-18 plus the roundings of x - m and of the result."""
import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import logprobs
from _layer_forms import HALF, TINY, TYPES, close, tokens as form

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
SHAPES = [(1, 1), (3, 2), (2, 7), (5, 8), (4, 33), (1, 1000), (300, 257), (7, 4097), (2, 32000), (1, 131072), (1, 131071), (40, 10001), (200, 2048), (700, 64)]


def make(rows, vocab, dtype, seed=0, size=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 65537 + rows * 257 + vocab)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * size).to(dtype)
    return x, torch.randint(0, vocab, (rows,), generator=g, device="cuda")


def floor(x):
    size = torch.where(torch.isfinite(x), x, 0).double().abs().amax(-1)
    return 2.0 ** -18 + 4 * F32 * size


def order(x, top):
    v, i = torch.sort(torch.where(torch.isnan(x), float("inf"), x.float()).double() + 0.0, dim=-1, descending=True, stable=True)
    return i[..., :top]


def check(x, ids, top, ignore=-100):
    r = logprobs.token_logprobs(x, ids, top=top, ignore_index=ignore)
    lp, entropy, logs = form(x, ids, ignore)
    f = floor(x)
    close(r.logprob, lp, 2 * F32, f)
    close(r.entropy, entropy, 2.0 ** -18, 4 * f)
    if top:
        want = order(x, top)
        assert r.top_tokens.dtype == torch.int64 and torch.equal(r.top_tokens, want)
        close(r.top_logprobs, logs.gather(-1, want), 2 * F32, f[..., None])
    else:
        assert r.top_logprobs is None and r.top_tokens is None
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, vocab", SHAPES)
def test_forward(rows, vocab, dtype):
    x, ids = make(rows, vocab, dtype)
    for top in {0, 1, min(5, vocab), min(20, vocab), min(32, vocab)}:
        r = check(x, ids, top)
        s = logprobs.token_logprobs(x, ids, top=top)
        assert all(p is None and q is None or torch.equal(p, q) for p, q in zip(r, s))
    none = logprobs.token_logprobs(x)
    assert none.logprob is None and torch.equal(none.entropy, logprobs.token_logprobs(x, ids).entropy)


@pytest.mark.parametrize("pattern", ["rising", "falling", "equal", "two values", "one peak", "zeros", "sawtooth"])
@pytest.mark.parametrize("vocab", [40, 1000, 50001])
def test_orders_and_ties(pattern, vocab):
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    x = {"rising": i / vocab, "falling": -i / vocab, "equal": torch.zeros(vocab, device="cuda"), "two values": (i % 3 == 1).float(),
         "one peak": torch.where(i == vocab // 2, 60.0, 0.0), "zeros": torch.where(i % 2 == 0, -0.0, 0.0), "sawtooth": i % 37}[pattern]
    x = torch.stack([x, x.flip(0), x.roll(5)])
    check(x, torch.tensor([0, vocab // 2, vocab - 1], device="cuda"), 32)
    check(x.bfloat16(), torch.tensor([0, vocab // 2, vocab - 1], device="cuda"), 7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [33, 5000, 40001])
def test_masks(vocab, dtype):
    x, ids = make(9, vocab, dtype, 1)
    x[0, :] = -float("inf")                       # nothing left
    x[1, :-1] = -float("inf")                     # one left, the last
    ids[1] = vocab - 1
    x[2, 1:] = -float("inf")                      # the first
    x[3, ids[3]] = -float("inf")                  # the token itself is masked
    x[4, : vocab // 2] = -float("inf")
    x[5] = torch.finfo(dtype).min                 # a mask of the type's lowest value in every place
    x[6, 1::2] = torch.finfo(dtype).min
    x[7, :20] = -float("inf")
    r = check(x, ids, 32)
    assert r.logprob[0] == -float("inf") and r.entropy[0] == 0 and torch.equal(r.top_tokens[0], torch.arange(32, device="cuda"))
    assert r.logprob[1] == 0 and r.entropy[1] == 0
    y = x.detach().requires_grad_(True)
    lp, h = tp.token_logprobs(y, ids)
    (g,) = torch.autograd.grad((lp, h), y, (torch.ones_like(lp), torch.ones_like(h)))
    assert not g[0].any() and torch.isfinite(g[torch.arange(9) != 3]).all() and not g[torch.isinf(x)][: 33].any()


def test_rows_that_are_not_finite():
    for vocab in (40, 5000, 40001):
        x, ids = make(6, vocab, torch.float32, 2)
        x[1, 3], x[2, vocab - 1], x[4, 0] = float("nan"), float("inf"), float("nan")
        x[4, 1:] = -float("inf")
        y = x.requires_grad_(True)
        r = logprobs.token_logprobs(x, ids, top=3)
        for t in (r.logprob, r.entropy, r.top_logprobs):
            assert torch.isnan(t[[1, 2, 4]]).all() and torch.isfinite(t[[0, 3, 5]]).all()
        assert r.top_tokens[1, 0] == 3 and r.top_tokens[2, 0] == vocab - 1
        assert ((r.top_tokens >= 0) & (r.top_tokens < vocab)).all()
        lp, h = tp.token_logprobs(y, ids)
        (g,) = torch.autograd.grad(lp.sum(), y)
        assert torch.isnan(g[[1, 2, 4]]).all() and torch.isfinite(g[[0, 3, 5]]).all()


def test_tokens_that_are_none():
    x, ids = make(6, 300, torch.float32, 3)
    ids[0], ids[1], ids[2], ids[3] = -100, 300, -1, 2 ** 40
    x.requires_grad_(True)
    r = logprobs.token_logprobs(x, ids)
    assert r.logprob[0] == 0 and torch.isnan(r.logprob[1:4]).all() and torch.isfinite(r.logprob[4:]).all() and torch.isfinite(r.entropy).all()
    (g,) = torch.autograd.grad(tp.token_logprobs(x, ids)[0].sum(), x)
    assert not g[0].any() and torch.isnan(g[1:4]).all() and torch.isfinite(g[4:]).all()
    (g,) = torch.autograd.grad(tp.token_logprobs(x, ids)[1].sum(), x)   # entropies need no token
    assert torch.isfinite(g).all() and g[0].any()
    assert logprobs.token_logprobs(x, ids, ignore_index=300).logprob[1] == 0
    assert not torch.isnan(logprobs.token_logprobs(x, torch.full_like(ids, 7), ignore_index=7).logprob).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, vocab", SHAPES)
def test_gradient(rows, vocab, dtype):
    x, ids = make(rows, vocab, dtype, 4)
    x.requires_grad_(True)
    gl, gh = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    if rows > 2:
        ids[rows // 2] = -100
    lp, h = tp.token_logprobs(x, ids)
    for take, grads in (((lp, h), (gl, gh)), ((lp,), (gl,)), ((h,), (gh,))):
        (g,) = torch.autograd.grad(take, x, grads, retain_graph=True)
        _, entropy, logs = form(x.detach(), ids)
        p = logs.exp()
        a = torch.where(ids == -100, 0.0, gl.double())[:, None] if len(take) == 2 or take[0] is lp else torch.zeros(rows, 1, device="cuda", dtype=torch.float64)
        b = gh.double()[:, None] if len(take) == 2 or take[0] is h else torch.zeros_like(a)
        want = -a * p - b * p * (logs + entropy[:, None])
        want.scatter_add_(1, torch.where(ids == -100, 0, ids)[:, None], a)
        f = floor(x.detach())[:, None]
        close(g, want, 1.01 * HALF[dtype], (a.abs() * 2 + b.abs() * (2 + logs.abs() + entropy[:, None])) * (p * 8 * f + 2 * F32 * (want != 0)) + TINY[dtype])


def test_gradient_against_differences():
    x = torch.randn(2, 12, device="cuda", requires_grad=True)
    ids, gl, gh = torch.tensor([3, 11], device="cuda"), torch.tensor([1.0, -0.5], device="cuda"), torch.tensor([0.7, 2.0], device="cuda")
    (g,) = torch.autograd.grad(tp.token_logprobs(x, ids), x, (gl, gh))
    want = torch.empty_like(g)
    with torch.no_grad():
        for i in range(2):
            for j in range(12):
                v = []
                for d in (2.0 ** -6, -(2.0 ** -6)):
                    y = x.detach().clone()
                    y[i, j] += d
                    r = logprobs.token_logprobs(y, ids)
                    v.append(float((r.logprob.double() * gl).sum() + (r.entropy.double() * gh).sum()))
                want[i, j] = (v[0] - v[1]) / 2 ** -5
    assert float((g - want).norm() / want.norm()) < 1e-3   # second order: (2^-6)^2 / 6 of third derivatives of size one, and f32 steps of 2^-22 over 2^-5


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(dtype):
    wide, ids = make(24, 1300, dtype, 5)
    for skip in (0, 1, 3, 8):
        x = wide[:, skip:skip + 1201]
        want, got = logprobs.token_logprobs(x.contiguous(), ids % 1201, top=4), logprobs.token_logprobs(x, ids % 1201, top=4)
        assert torch.equal(want.top_tokens, got.top_tokens)
        close(got.logprob, want.logprob.double(), 2 * F32, 2 * floor(x))
        g1 = logprobs.token_logprobs_backward(x, ids % 1201, got.stats, got.entropy, torch.ones(24, device="cuda"), torch.ones(24, device="cuda"))
        g2 = logprobs.token_logprobs_backward(x.contiguous(), ids % 1201, got.stats, got.entropy, torch.ones(24, device="cuda"), torch.ones(24, device="cuda"))
        assert torch.equal(g1, g2)
    x3 = wide.view(2, 12, 1300)
    r = logprobs.token_logprobs(x3, ids.view(2, 12), top=3)
    assert r.logprob.shape == (2, 12) and r.top_tokens.shape == (2, 12, 3) and r.stats.shape == (2, 12, 2)
    assert torch.equal(r.logprob.view(-1), logprobs.token_logprobs(wide, ids).logprob)
    one = logprobs.token_logprobs(wide[0], ids[0], top=2)
    assert one.logprob.shape == () and one.top_tokens.shape == (2,)
    assert logprobs.token_logprobs(wide[:0], ids[:0], top=2).top_tokens.shape == (0, 2)
    columns = wide.t()[:24].contiguous().t()
    assert torch.equal(logprobs.token_logprobs(columns, top=2).top_tokens, logprobs.token_logprobs(columns.contiguous(), top=2).top_tokens)


def test_other_streams_and_capture():
    x, ids = make(30, 9000, torch.bfloat16, 6)
    x.requires_grad_(True)
    gl = torch.randn(30, device="cuda")

    def step():
        lp, h = tp.token_logprobs(x, ids)
        return [lp.detach(), h.detach(), *torch.autograd.grad((lp, h), x, (gl, gl)), *logprobs.token_logprobs(x, ids, top=9)[:4]]

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
