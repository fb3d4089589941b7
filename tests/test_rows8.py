"""8-bit rows without a GPU: refusals of the Python surface and of the C ABI."""
import os
import subprocess

import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import _native as N
from tropical_gemm import rows8
from tropical_gemm.rows8 import Rows8

F32, F64, I32, BF16, F16 = 0, 1, 2, 4, 5
P = 0x1000   # a pointer that validation never follows


def r8(*shape):
    return Rows8(torch.zeros(*shape, dtype=torch.int8), torch.zeros(*shape[:-1]))


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8)
    for call in (lambda: rows8.quantize(x), lambda: rows8.dequantize(r8(2, 8)), lambda: rows8.rmsnorm(x, torch.ones(8)),
                 lambda: rows8.matmul(r8(2, 8), r8(3, 8)), lambda: rows8.matmul_backward(x, None, r8(8, 4)),
                 lambda: rows8.rmsnorm_backward(x, r8(2, 8), torch.zeros(2), torch.ones(8)), lambda: rows8.column_sum(x),
                 lambda: tp.rmsnorm_linear_rows8(x, torch.ones(8), torch.zeros(4, 8))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("call", [
    lambda: rows8.quantize(torch.zeros(2, 8, dtype=torch.float64)),
    lambda: rows8.quantize(torch.zeros(2, 8, dtype=torch.int8)),
    lambda: rows8.dequantize(Rows8(torch.zeros(2, 8), torch.zeros(2))),
    lambda: rows8.dequantize(Rows8(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(3))),
    lambda: rows8.matmul(Rows8(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2, dtype=torch.float64)), r8(3, 8)),
    lambda: rows8.matmul_backward(torch.zeros(2, 3, dtype=torch.int32), None, r8(3, 8)),
    lambda: tp.rmsnorm_linear_rows8(torch.zeros(2, 8), torch.ones(8), torch.zeros(4, 8, dtype=torch.bfloat16)),
])
def test_wrong_types_are_value_errors(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("name, args, code", [
    ("tg_rows8_quantize", (F64, 2, 8, P, 8, P, 8, P, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_quantize", (9, 2, 8, P, 8, P, 8, P, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_quantize", (F32, -1, 8, P, 8, P, 8, P, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_quantize", (F32, 2, 8, None, 8, P, 8, P, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_quantize", (F32, 2, 8, P, 7, P, 8, P, None), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_rows8_quantize", (F32, 2, 8, P, 8, P, 7, P, None), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_rows8_dequantize", (I32, 2, 8, P, 8, P, P, 8, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_dequantize", (BF16, 2, 8, P, 8, P, P, 5, None), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_rows8_rmsnorm", (BF16, 2, 8, P, 8, None, 0, P, -1.0, None, 8, P, 8, P, None, 8, None, None, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_rmsnorm", (BF16, 2, 8, P, 8, None, 0, P, 0.0, None, 8, P, 8, P, P, 8, None, None, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_rmsnorm", (BF16, 2, 8, P, 8, P, 4, P, 0.0, None, 8, P, 8, P, None, 8, None, None, None), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_rows8_rmsnorm", (BF16, 2, 8, P, 8, None, 0, None, 0.0, None, 8, P, 8, P, None, 8, None, None, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_rmsnorm_backward", (BF16, F16, 2, 8, P, 8, None, 0, P, P, 8, P, P, P, 8, P, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_rmsnorm_backward", (BF16, F32, 2, 8, P, 8, None, 0, P, P, 3, P, P, P, 8, P, None), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_rows8_rmsnorm_backward", (BF16, F32, 2, 8, P, 8, None, 0, P, None, 8, P, P, P, 8, P, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_gemm", (F64, 4, 4, 4, P, 4, P, P, 4, P, None, P, 4, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_gemm", (F32, 4, -4, 4, P, 4, P, P, 4, P, None, P, 4, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_gemm", (F32, 4, 4, 4, P, 4, None, P, 4, P, None, P, 4, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_gemm", (F32, 4, 4, 4, P, 3, P, P, 4, P, None, P, 4, None), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_rows8_gemm", (F32, 4, 4, 4, P, 4, P, P, 4, P, None, P, 3, None), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_rows8_gemm", (F32, 4, 4, 1 << 17, P, 1 << 17, P, P, 1 << 17, P, None, P, 4, None), N.TG_ERR_UNSUPPORTED),
    ("tg_rows8_gemm_backward", (F64, F32, 0, 4, 4, 4, P, 4, P, 4, P, P, 4, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_gemm_backward", (F32, I32, 0, 4, 4, 4, P, 4, P, 4, P, P, 4, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_gemm_backward", (F32, F32, 1, 8, 4, 4, P, 4, P, 4, P, P, 4, None), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_rows8_gemm_backward", (F32, F32, 0, 4, 4, 4, P, 4, P, 4, None, P, 4, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_column_sum", (F32, F64, 4, 4, P, 4, P, None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_rows8_column_sum", (F32, F32, 4, 4, P, 2, P, None), N.TG_ERR_DIMENSION_MISMATCH),
])
def test_abi_refusals(name, args, code):
    L = N.lib()
    assert getattr(L, name)(*args) == code
    assert len(L.tg_last_error()) > 0


def test_empty_problems_touch_nothing():
    L = N.lib()
    assert L.tg_rows8_quantize(F32, 0, 8, None, 8, None, 8, None, None) == N.TG_OK
    assert L.tg_rows8_dequantize(F32, 3, 0, None, 0, None, None, 0, None) == N.TG_OK
    assert L.tg_rows8_gemm(F32, 0, 4, 4, None, 4, None, None, 4, None, None, None, 4, None) == N.TG_OK
    assert L.tg_rows8_gemm_backward(F32, F32, 0, 4, 0, 4, None, 4, None, 0, None, None, 0, None) == N.TG_OK


def test_tropical_calls_refuse_the_16_bit_types():
    L = N.lib()
    for t in (BF16, F16):
        assert L.tg_gemm(0, t, 0, 4, 4, 4, P, 4, P, 4, P, 4, None, None) == N.TG_ERR_INVALID_ARGUMENT
        assert L.tg_backward_a(0, t, 0, 1, 4, 4, 4, P, 4, 16, P, None, 4, 16, P, 4, 16, 0, None) == N.TG_ERR_UNSUPPORTED


@pytest.mark.parametrize("m, n", [(1, 0x7ffffc01), (64, 1 << 31), (40, 1 << 34), (0x7ffffc01, 16), (1 << 33, 16)])
@pytest.mark.parametrize("ld", [16, 24])
def test_products_of_too_many_rows_or_columns_are_refused(m, n, ld):
    """Whatever kernel the number of tokens would take, and before any scratch or launch."""
    L = N.lib()
    assert L.tg_rows8_gemm(BF16, m, n, 16, P, ld, P, P, ld, P, None, P, n, None) == N.TG_ERR_UNSUPPORTED
    assert b"outputs" in L.tg_last_error()


def test_the_library_builds_without_torch():
    """The C library and its probe need nvcc alone; the torch binding is a target of its own."""
    def commands(*target):
        pkg = os.path.dirname(os.path.dirname(os.path.abspath(N.__file__)))
        return subprocess.run(["make", "-n", "-B", "-C", pkg, "PYTHON=no-such-python", *target], check=True, capture_output=True, text=True).stdout

    assert "libtropical_gemm_b200.so" in commands() and "rows8_torch" not in commands() and "no-such-python" not in commands()
    assert "rows8_torch" in commands("torch") and "libtropical_gemm_b200.so" in commands("torch")
