"""8-bit rows on the GPU: calls at the ends of their ranges."""
import pytest
import torch

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
