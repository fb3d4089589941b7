"""Layer norm of finite rows whose sums or squares pass f32's range: statistics that are finite, and neighbours left alone.

The mean is a sum of h / cols: cols additions of at most half a step of the largest |h| each, in a tree of a few dozen, and the
rounding of 1 / cols: 64 half steps of the largest |h|."""
import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import blocks8, norms
from _layer_forms import HALF, close, norm

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
COLS = [8, 512, 1001, 4608, 8192, 20000]


def rows_of(cols, dtype):
    """Ordinary rows 0, 2, 5 and 8; between them normal ones of 1e20, 1e28 and 1e36, one of 1e36 throughout, half 1e36 and half -1e36, 2^126 throughout."""
    x = torch.randn(9, cols, device="cuda")
    far = [1, 3, 4, 6, 7]
    x[1] *= 1e28
    x[3] *= 1e36
    x[4] = 1e36
    x[6] = torch.where(torch.arange(cols, device="cuda") * 2 < cols, 1e36, -1e36)
    x[7] = 2.0 ** 126
    return x.to(dtype), far


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", COLS)
def test_far_rows(cols, dtype):
    x, far = rows_of(cols, dtype)
    w, b, g, gh = (torch.randn(s, device="cuda").to(dtype) for s in ((cols,), (cols,), (9, cols), (9, cols)))
    r = norms.layernorm(x, w, b, stats=True)
    close(r.mean, x.double().mean(-1), F32, 64 * F32 * x.double().abs().amax(-1))
    for i in far:
        if float((x[i].double() - x[i].double().mean()).square().sum()) > 1e39:   # f32 ends at 3.4e38
            assert r.rstd[i] == 0
        if r.rstd[i] == 0:
            assert torch.equal(r.y[i], b)
    assert torch.isfinite(r.y).all() and torch.isfinite(r.rstd).all() and (r.rstd[far] < 1e-9).sum() >= 3
    near = [0, 2, 5, 8]
    alone = norms.layernorm(torch.where(torch.isin(torch.arange(9, device="cuda"), torch.tensor(near, device="cuda"))[:, None], x, 0.0), w, b, stats=True)
    assert torch.equal(r.y[near], alone.y[near])
    gx, gw, gb = norms.layernorm_backward(g, x, r.mean, r.rstd, w, gh)
    zero = r.rstd == 0
    assert torch.equal(gx[zero], gh[zero]) and torch.isfinite(gx).all()
    h, u, rstd, _ = norm(x[near])   # far rows: rstd is 0, or, where all values are the same, their distance
    size = (1 + u.abs().amax(-1, keepdim=True)) * (1 + h.abs().amax(-1, keepdim=True) * rstd / 8) + u.abs()
    close(gw, (g[near].double() * u).sum(0), 1.01 * HALF[dtype], 64 * F32 * (g[near].double().abs() * size).sum(0))
    n = blocks8.layernorm(x, w, b)
    assert torch.isfinite(n.blocks.scale).all()


@pytest.mark.parametrize("cols", COLS)
def test_training_beside_a_far_row(cols):
    x, far = rows_of(cols, torch.float32)
    x.requires_grad_(True)
    w = torch.randn(cols, device="cuda", requires_grad=True)
    y, _ = tp.layernorm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.randn_like(y))
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all()


def test_a_row_at_the_end_of_squares():
    """1e18 over 64 columns: squares add up to 6.4e37, within range, and the row has its norm."""
    x = torch.randn(4, 64, device="cuda") * 1e18
    r = norms.layernorm(x, stats=True)
    _, u, rstd, _ = norm(x)
    close(r.rstd, rstd[:, 0], 64 * F32)
    close(r.y, u, F32, 64 * F32 * float(u.abs().max() + 1))


@pytest.mark.parametrize("cols", COLS)
def test_infinities_and_nan_stay(cols):
    x = torch.randn(7, cols, device="cuda")
    x[1, cols // 2], x[3, 0], x[4, cols - 1] = float("nan"), float("inf"), -float("inf")
    x[5] = float("inf")
    r = norms.layernorm(x, stats=True)
    assert torch.isnan(r.y[[1, 3, 4, 5]]).all() and torch.isfinite(r.y[[0, 2, 6]]).all()
    assert torch.isnan(r.rstd[[1, 3, 4, 5]]).all()
