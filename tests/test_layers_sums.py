"""The layer norm's backward of sums without a GPU: refusals of the Python surface and of the C ABI."""
import pytest
import torch

from tropical_gemm import _native as N
from tropical_gemm import norms

P = 0x1000   # a pointer that validation never follows
F16 = 5
CALL = (F16, 2, 8, P, 8, None, 0, P, P, 8, P, 8, P, P, P, 8, P, P, None)


def but(**at):
    return tuple(at.get(f"a{i}", v) for i, v in enumerate(CALL))


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        norms.layernorm_backward(x, x, torch.zeros(2), torch.zeros(2), residual=x)


@pytest.mark.parametrize("args, code", [
    (but(a0=1), N.TG_ERR_INVALID_ARGUMENT), (but(a1=-1), N.TG_ERR_INVALID_ARGUMENT), (but(a2=0), N.TG_ERR_INVALID_ARGUMENT), (but(a3=None), N.TG_ERR_INVALID_ARGUMENT),
    (but(a8=None), N.TG_ERR_INVALID_ARGUMENT), (but(a12=None), N.TG_ERR_INVALID_ARGUMENT), (but(a13=None), N.TG_ERR_INVALID_ARGUMENT),
    (but(a4=7), N.TG_ERR_DIMENSION_MISMATCH), (but(a5=P, a6=7), N.TG_ERR_DIMENSION_MISMATCH), (but(a9=7), N.TG_ERR_DIMENSION_MISMATCH),
    (but(a11=7), N.TG_ERR_DIMENSION_MISMATCH), (but(a15=7), N.TG_ERR_DIMENSION_MISMATCH), (but(a2=1 << 31), N.TG_ERR_UNSUPPORTED),
])
def test_abi_refusals(args, code):
    L = N.lib()
    assert L.tg_layernorm_residual_backward(*args) == code
    assert len(L.tg_last_error()) > 0


def test_empty_problems_touch_nothing():
    L = N.lib()
    assert L.tg_layernorm_residual_backward(*but(a14=None, a16=None, a17=None)) == N.TG_OK
    assert L.tg_layernorm_residual_backward(*but(a1=0, a3=None, a8=None, a16=None, a17=None)) == N.TG_OK
