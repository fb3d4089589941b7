"""The inner loops that large calls of the layers run: stages and slots used again, several warps and batches of a row's alternatives, rows
and launches after the first; and what calls leave alone.

Tolerances are those of the layers' own tests: test_gpu_layernorm_sums.check, test_gpu_logprobs.check."""
import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import blocks8, logprobs, norms
from tropical_gemm.blocks8 import Blocks8
from _layer_forms import HALF, TINY, TYPES, close, tokens as form
from test_gpu_layernorm_sums import check as check_gradients
from test_gpu_logprobs import check as check_tokens, floor

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24


def normal(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + sum(shape))
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# ---------------------------------------------------------------------------------------------------------------- layer norm
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols, skip", [(2400, 8192, 0), (2400, 4096, 8), (2401, 4099, 0), (1900, 6001, 3), (9000, 250, 0), (12000, 128, 0), (5000, 1000, 1)])
def test_norm_backward_of_many_rows(rows, cols, skip, dtype):
    """More rows to a block than its ring has stages: on 148 SMs 16 rows each of 2400, and 8 stages at most.  Rows that start on a boundary, all
    at the same distance from one, and each operand at another."""
    x, g, gh = (normal(rows, cols + 2 * skip, dtype=dtype, seed=i)[:, skip * (i != 1):][:, :cols] for i in range(3))
    w = (1 + 0.2 * normal(cols)).to(dtype)
    f = norms.layernorm(x, w, stats=True)
    for weight, grad_h in ((w, gh), (None, None)):
        got = norms.layernorm_backward(g, x, f.mean, f.rstd, weight, grad_h)
        check_gradients(got, x, None, weight, g, grad_h)
        assert all(torch.equal(p, q) for p, q in zip(got, norms.layernorm_backward(g, x, f.mean, f.rstd, weight, grad_h)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, cols, pad, skip", [(5, 64, 3, 1), (40, 257, 8, 8), (9, 1000, 5, 2), (600, 130, 2, 6), (300, 4100, 1, 5), (3, 20000, 1, 1)])
def test_wider_matrices_are_left_alone(rows, cols, pad, skip, dtype):
    """Rows of wider matrices: nothing of them, or beside them, is written."""
    wide = [normal(rows, cols + pad + skip + 16, dtype=dtype, seed=i) for i in range(4)]
    before = [t.clone() for t in wide]
    x, res, g, gh = (t[:, skip + i:skip + i + cols] for i, t in enumerate(wide))
    w, b = (normal(cols + 1, dtype=dtype, seed=i)[1:] for i in range(2))
    kept = w.clone(), b.clone()
    f = norms.layernorm(x, w, b, residual=res, stats=True)
    norms.layernorm_backward(g, x, f.mean, f.rstd, w, gh)
    norms.layernorm_backward(g, x, f.mean, f.rstd, w, gh, residual=res)
    blocks8.layernorm(x, w, b, residual=res)
    blocks8.quantize_both(x)
    blocks8.quantize_tiles(x)
    r = logprobs.token_logprobs(x, top=3)
    logprobs.token_logprobs_backward(x, None, r.stats, r.entropy, None, torch.ones(rows, device="cuda"))
    assert all(torch.equal(s, t) for s, t in zip(wide, before)) and torch.equal(w, kept[0]) and torch.equal(b, kept[1])


def test_h_has_no_part_in_the_weights_gradient():
    x, w, b, g, gh = normal(5, 40), normal(40, seed=1), normal(40, seed=2), normal(5, 40, seed=3), normal(5, 40, seed=4)
    w.requires_grad_(True)
    for res in (None, normal(5, 40, seed=5)):
        y, h = tp.layernorm(x, w, b, residual=res)
        (alone,) = torch.autograd.grad(y, w, g, retain_graph=True)
        (both,) = torch.autograd.grad((y, h), w, (g, gh), retain_graph=True)
        assert torch.equal(alone, both)
        assert torch.autograd.grad(h, w, gh, allow_unused=True) == (None,)


# ------------------------------------------------------------------------------------------------------- log probabilities
def logits(pattern, rows, vocab, dtype):
    if pattern == "normal":
        return (3 * normal(rows, vocab)).to(dtype)
    rise = torch.arange(vocab, device="cuda", dtype=torch.float32) / vocab
    x = {"rising": rise, "falling": -rise, "sawtooth": torch.arange(vocab, device="cuda") % 1021 / 1021.0}[pattern]
    return (x[None] + normal(rows, 1)).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pattern", ["normal", "rising", "falling", "sawtooth"])
@pytest.mark.parametrize("rows, vocab, tops", [(500, 20001, (1, 5, 20, 32)), (500, 40000, (20,)), (800, 20000, (0,)), (1500, 5003, (0, 32))])
def test_many_rows_of_many_logits(rows, vocab, tops, pattern, dtype):
    """From three rows per SM on with alternatives and five without, a row has four warps, and 4096 logits go into a batch."""
    x = logits(pattern, rows, vocab, dtype)
    ids = torch.randint(0, vocab, (rows,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for top in tops:
        check_tokens(x, ids, top)


@pytest.mark.parametrize("dtype", TYPES)
def test_masks_among_many_rows(dtype):
    rows, vocab = 600, 20001
    x = logits("normal", rows, vocab, dtype)
    ids = torch.randint(0, vocab, (rows,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    x[0::7] = -float("inf")                    # nothing left
    x[1::7, 5000:] = -float("inf")             # the first batch alone
    x[2::7, :17000] = -float("inf")            # the last alone
    x[3::7, 40:] = -float("inf")               # about as many as alternatives
    x[4::7] = torch.finfo(dtype).min
    x[5::7, 1::2] = torch.finfo(dtype).min
    check_tokens(x, ids, 32)
    y = x.clone()
    y[0::7, 9000], y[1::7, 3], y[6::7, 20000] = float("nan"), float("inf"), float("nan")
    r = logprobs.token_logprobs(y, ids, top=20)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[0::7] = bad[1::7] = bad[6::7] = True
    same = logprobs.token_logprobs(x, ids, top=20)
    for p, q in zip(r, same):
        assert torch.equal(p[~bad], q[~bad])
    assert torch.isnan(r.logprob[bad]).all() and torch.isnan(r.entropy[bad]).all() and torch.isnan(r.top_logprobs[bad]).all()
    assert (r.top_tokens[0::7, 0] == 9000).all() and (r.top_tokens[1::7, 0] == 3).all() and (r.top_tokens[6::7, 0] == 20000).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, vocab, top", [(70000, 40, 5), (70000, 41, 32), (66000, 1300, 3), (66000, 1300, 0)])
def test_rows_taken_in_turn(rows, vocab, top, dtype):
    """Beyond 65536 rows a block takes another one: no bound, list or sum of the last row's is left in it."""
    x = logits("normal", rows, vocab, dtype)
    x[65536:] -= 20   # below all that the first rows' lists and bounds held
    ids = torch.randint(0, vocab, (rows,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    check_tokens(x, ids, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, vocab", [(1500, 9000), (4000, 301), (300, 40001)])
def test_gradients_of_many_rows(rows, vocab, dtype):
    """More rows, or parts of rows, than blocks: eight per SM, 1184 on 148."""
    x = logits("normal", rows, vocab, dtype).requires_grad_(True)
    ids = torch.randint(0, vocab, (rows,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    ids[5::11] = -100
    gl, gh = normal(rows), normal(rows, seed=1)
    lp, h = tp.token_logprobs(x, ids)
    (g,) = torch.autograd.grad((lp, h), x, (gl, gh))
    _, entropy, logs = form(x.detach(), ids)
    p = logs.exp()
    a, b = torch.where(ids == -100, 0.0, gl.double())[:, None], gh.double()[:, None]
    want = -a * p - b * p * (logs + entropy[:, None])
    want.scatter_add_(1, torch.where(ids == -100, 0, ids)[:, None], a)
    f = floor(x.detach())[:, None]
    close(g, want, 1.01 * HALF[dtype], (a.abs() * 2 + b.abs() * (2 + logs.abs() + entropy[:, None])) * (p * 8 * f + 2 * F32 * (want != 0)) + TINY[dtype])


# ------------------------------------------------------------------------------------------------------------- 8-bit blocks
def same_codes(a, b):
    return torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scale, b.scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [8, 13])
def test_more_rows_of_tiles_than_one_launch_takes(cols, dtype):
    """32768 rows of tiles go into a launch: a matrix of 300 rows more is as its two halves are."""
    rows, half = 32768 * 128 + 300, 16384 * 128
    x = normal(rows, cols, dtype=dtype)
    parts = [x[:half], x[half:2 * half], x[2 * half:]]
    whole, turned = blocks8.quantize_both(x)
    a = [blocks8.quantize_both(p) for p in parts]
    cat = lambda ts, d=0: torch.cat([t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in ts], d)   # noqa: E731
    assert torch.equal(whole.q.view(torch.uint8), cat([p.q for p, _ in a])) and torch.equal(whole.scale, cat([p.scale for p, _ in a]))
    assert torch.equal(turned.q.contiguous().view(torch.uint8), cat([t.q.contiguous() for _, t in a], 1)) and torch.equal(turned.scale, cat([t.scale for _, t in a], 1))
    assert same_codes(blocks8.quantize(x), whole)
    tiles, b = blocks8.quantize_tiles(x), [blocks8.quantize_tiles(p) for p in parts]
    assert torch.equal(tiles.q.view(torch.uint8), cat([p.q for p in b])) and torch.equal(tiles.scale, cat([p.scale for p in b]))


def test_bias_gradient_of_more_rows_than_one_launch_takes():
    rows = 32768 * 128 + 300
    x, w, b = torch.zeros(rows, 8, device="cuda"), normal(8, 8), torch.zeros(8, device="cuda", requires_grad=True)
    g = torch.randint(-3, 4, (rows, 8), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).float()
    (gb,) = torch.autograd.grad(tp.linear_blocks8(x, w, b), b, g)
    assert torch.equal(gb.long(), g.long().sum(0))   # whole numbers below 2^24: exact in any order


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, n", [(1, 8), (127, 40), (3000, 257), (700, 4096)])
def test_bias_gradient(rows, n, dtype):
    """Rows of one size: f32 sums, at most 64 additions deep, and one rounding."""
    x, w, b, g = normal(rows, 24, dtype=dtype), normal(n, 24, dtype=dtype), normal(n, dtype=dtype).requires_grad_(True), normal(rows, n, dtype=dtype, seed=1)
    (gb,) = torch.autograd.grad(tp.linear_blocks8(x, w, b), b, g)
    close(gb, g.double().sum(0), 1.01 * HALF[dtype], 64 * F32 * g.double().abs().sum(0) + TINY[dtype])


# ------------------------------------------------------------------------------------------ offsets that pass 32 bits
def test_more_than_two_to_the_31_elements():
    """Rows far into a tensor are as they are alone.  70000 x 32768, 4.3 GiB; the slice has its own many rows, so that the same kernels take it."""
    rows, cols, last = 70000, 32768, 2000
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for i in range(0, rows, 10000):
        x[i:i + 10000] = normal(10000, cols, dtype=torch.bfloat16, seed=i)
    tail = x[rows - last:].clone()
    ids = torch.arange(rows, device="cuda") % cols
    r, s = logprobs.token_logprobs(x, ids, top=4), logprobs.token_logprobs(tail, ids[rows - last:], top=4)
    assert all(torch.equal(p[rows - last:], q) for p, q in zip(r, s))
    one = torch.ones(rows, device="cuda")
    g = logprobs.token_logprobs_backward(x, ids, r.stats, r.entropy, one, one)[rows - last:].clone()
    assert torch.equal(g, logprobs.token_logprobs_backward(tail, ids[rows - last:], s.stats, s.entropy, one[:last], one[:last]))
    del r, g
    for c in (cols, 4096):   # a row too long for registers, and eight times as many shorter ones
        v, t = x.view(-1, c), tail.view(-1, c)
        n = t.size(0)
        a, b = norms.layernorm(v, residual=v, stats=True), norms.layernorm(t, residual=t, stats=True)
        assert torch.equal(a.y[-n:], b.y) and torch.equal(a.h[-n:], b.h) and torch.equal(a.rstd[-n:], b.rstd)
        p = norms.layernorm_backward(v, v, a.mean, a.rstd, None, v, residual=v)[0][-n:].clone()
        assert torch.equal(p, norms.layernorm_backward(t, t, b.mean, b.rstd, None, t, residual=t)[0])
        del a, b, p
    e, f = blocks8.layernorm(x).blocks, blocks8.layernorm(tail).blocks
    assert torch.equal(e.q[rows - last:].view(torch.uint8), f.q.view(torch.uint8)) and torch.equal(e.scale[rows - last:], f.scale)
    a, t = blocks8.quantize_both(x)
    b = blocks8.quantize(tail)
    assert torch.equal(a.q[rows - last:].view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scale[rows - last:], b.scale)
    half = rows // 2 // 128 * 128
    u = blocks8.quantize_both(x[half:])[1]
    assert torch.equal(t.q[:, half:].contiguous().view(torch.uint8), u.q.contiguous().view(torch.uint8)) and torch.equal(t.scale[:, half // 128:], u.scale)
    w = blocks8.quantize_tiles(torch.eye(128, cols, device="cuda"))
    z = blocks8.matmul(a, w)
    assert torch.equal(z[rows - last:], blocks8.matmul(b, w))
    turned = blocks8.transpose(Blocks8(a.q, torch.ones(-(-rows // 128), cols // 128, device="cuda")))
    assert torch.equal(turned.q[-300:, -300:].float(), a.q[-300:, -300:].float().t())
    d = blocks8.dequantize(a)
    assert torch.equal(d[rows - last:], blocks8.dequantize(b))
