"""8-bit rows on the GPU: calls at the ends of their ranges."""
import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import _native as N
from tropical_gemm import rows8
from tropical_gemm.rows8 import Rows8

pytestmark = pytest.mark.gpu
CODES = {torch.float32: 0, torch.bfloat16: 4, torch.float16: 5}


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("f32_grad", [False, True])
@pytest.mark.parametrize("cols", [1, 8, 77, 4096, 33000])
def test_norm_backward_of_no_rows_needs_no_operands(dtype, f32_grad, cols):
    """With no rows every operand may be null: the weight's gradient is a sum of nothing."""
    out = torch.full((cols + 8,), 3.0, device="cuda", dtype=dtype)
    stream = torch.cuda.current_stream().cuda_stream
    code = CODES[dtype]
    N.check(N.lib().tg_rows8_rmsnorm_backward(code, 0 if f32_grad else code, 0, cols, None, cols, None, cols, None, None, cols,
                                              None, None, None, cols, out.data_ptr(), stream))
    assert not out[:cols].any() and (out[cols:] == 3).all()


@pytest.mark.parametrize("cols", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31 - 24, 2 ** 31 - 33, 2 ** 31 - 40])
def test_dequantize_the_longest_rows(cols):
    """A row of as many columns as are accepted, of 8-element groups whose ends lie past 2^31 - 1."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    q = torch.empty(1, cols, device="cuda", dtype=torch.int8)
    ramp = torch.arange(1 << 20, device="cuda").remainder(251).sub(125).to(torch.int8)
    for at in range(0, cols, 1 << 20):
        q[0, at:at + (1 << 20)] = ramp[:min(1 << 20, cols - at)]
    y = rows8.dequantize(Rows8(q, torch.full((1,), 0.5, device="cuda")), torch.float16)
    for at in range(0, cols, 1 << 28):   # exact: codes of 8 bits, halved
        part = slice(at, min(at + (1 << 28), cols))
        assert torch.equal(y[:, part], q[:, part].half() * 0.5)


def test_calls_record_no_graph():
    """Only the autograd layer is differentiable; the calls below it return plain results for any arguments."""
    x, res, w, weight, bias = (torch.randn(*s, device="cuda").requires_grad_(True) for s in ((6, 32), (6, 32), (32,), (5, 32), (5,)))
    n = rows8.rmsnorm(x, w, residual=res, checkpoint=True)
    b = rows8.quantize(weight)
    z = rows8.matmul(n.rows, b, bias=bias, dtype=torch.float32)
    grads = rows8.matmul_backward(z, n.rows, b) + rows8.rmsnorm_backward(x, n.checkpoint, n.rstd, w, grad_h=res)
    for t in (n.h, n.rows.scale, n.checkpoint.scale, n.rstd, b.scale, z, rows8.column_sum(x), rows8.dequantize(b), *grads):
        assert not t.requires_grad and t.grad_fn is None
    assert rows8.rmsnorm(x, w).h is x or rows8.rmsnorm(x, w).h.data_ptr() == x.data_ptr()


@pytest.mark.parametrize("needed", [False, True])
def test_frozen_scales_take_no_gradient(needed):
    """A frozen weight is a constant, whatever its scale says."""
    x, w = torch.randn(4, 32, device="cuda", requires_grad=needed), rows8.quantize(torch.randn(8, 32, device="cuda"))
    scale = w.scale.clone().requires_grad_(True)
    norm = torch.ones(32, device="cuda")
    z, _ = tp.rmsnorm_linear_rows8(x, norm, Rows8(w.q, scale))
    assert torch.equal(z, tp.rmsnorm_linear_rows8(x, norm, w)[0]) and z.requires_grad == needed
    if needed:
        z.sum().backward()
        assert x.grad is not None and scale.grad is None
