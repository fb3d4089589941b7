"""Layer norm, 8-bit block layers and token log probabilities without a GPU: refusals of the Python surface and of the C ABI."""
import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import _native as N
from tropical_gemm import blocks8, logprobs, norms
from tropical_gemm.blocks8 import Blocks8

F32, F64, I32, BF16, F16 = 0, 1, 2, 4, 5
P = 0x1000   # a pointer that validation never follows
E4M3 = torch.float8_e4m3fn


def b8(n, k, tiles=False):
    return Blocks8(torch.zeros(n, k).to(E4M3), torch.zeros(-(-n // 128) if tiles else n, -(-k // 128)))


X, W, IDS = torch.zeros(2, 8), torch.ones(8), torch.zeros(2, dtype=torch.int64)


@pytest.mark.parametrize("call", [
    lambda: norms.layernorm(X, W, W), lambda: norms.layernorm_backward(X, X, torch.zeros(2), torch.zeros(2), W), lambda: tp.layernorm(X),
    lambda: blocks8.quantize(X), lambda: blocks8.quantize_both(X), lambda: blocks8.quantize_tiles(X), lambda: blocks8.transpose(b8(2, 8, True)),
    lambda: blocks8.dequantize(b8(2, 8)), lambda: blocks8.layernorm(X), lambda: blocks8.matmul(b8(2, 8), b8(3, 8)), lambda: tp.linear_blocks8(X, torch.zeros(4, 8)),
    lambda: tp.linear_blocks8(X, b8(4, 8, True)), lambda: logprobs.token_logprobs(X, IDS), lambda: tp.token_logprobs(X, IDS),
    lambda: logprobs.token_logprobs_backward(X, IDS, torch.zeros(2, 2)),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="CUDA"):
        call()


@pytest.mark.parametrize("call", [
    lambda: norms.layernorm(X.double()), lambda: norms.layernorm(X.int()), lambda: tp.layernorm(torch.zeros(2, 8, dtype=torch.complex64)),
    lambda: blocks8.quantize(X.double()), lambda: blocks8.quantize_tiles(X.to(torch.int8)), lambda: blocks8.dequantize(Blocks8(X, torch.zeros(2, 1))),
    lambda: blocks8.dequantize(Blocks8(X.to(torch.float8_e5m2), torch.zeros(2, 1))), lambda: blocks8.dequantize(Blocks8(X.to(E4M3), torch.zeros(2, 1, dtype=torch.float64))),
    lambda: blocks8.dequantize(Blocks8(X.to(E4M3), torch.zeros(2))), lambda: blocks8.dequantize(Blocks8(X.to(E4M3), torch.zeros(3, 1))),
    lambda: blocks8.dequantize(Blocks8(torch.zeros(2, 130).to(E4M3), torch.zeros(2, 1))), lambda: blocks8.transpose(b8(300, 8)),
    lambda: blocks8.matmul(b8(300, 8, True), b8(3, 8)), lambda: blocks8.matmul(b8(2, 8), Blocks8(torch.zeros(3, 8).to(E4M3), torch.zeros(2, 1))),
    lambda: tp.linear_blocks8(X, torch.zeros(4, 8, dtype=torch.bfloat16)), lambda: tp.linear_blocks8(X, torch.zeros(4, 9)), lambda: tp.linear_blocks8(X, torch.zeros(8)),
    lambda: tp.linear_blocks8(torch.zeros(()), torch.zeros(4, 8)), lambda: tp.linear_blocks8(X.double(), torch.zeros(4, 8, dtype=torch.float64)),
    lambda: logprobs.token_logprobs(X.double(), IDS),
])
def test_wrong_types_and_shapes_are_value_errors(call):
    with pytest.raises(ValueError):
        call()


NORM = (BF16, 2, 8, P, 8, None, 0, P, P, 1e-5, None, 8, P, 8, None, None, None)
NORM_BACK = (F16, 2, 8, P, 8, None, 0, P, P, 8, P, P, P, 8, P, P, None)
QUANT = (F32, 2, 8, P, 8, P, 8, P, 1, 2, None, 0, None, 0, 0, None, None)
TILES = (F32, 2, 8, P, 8, P, 8, P, 1, 1, None, 0, None)
VALUES = (F32, 2, 8, 1, P, 8, P, 1, 1, P, 8, None)
NORM8 = (BF16, 2, 8, P, 8, None, 0, P, P, 1e-5, None, 8, P, 8, P, 1, 2, None, None, None)
GEMM = (F32, 4, 4, 4, P, 4, P, 1, 1, P, 4, 128, P, 1, 1, None, P, 4, None)
TOKENS = (BF16, 2, 8, P, 8, P, -100, P, P, P, 2, P, P, None)
TOKENS_BACK = (BF16, 2, 8, P, 8, P, -100, P, P, P, P, P, 8, None)


def but(args, **at):
    return tuple(at.get(f"a{i}", v) for i, v in enumerate(args))


@pytest.mark.parametrize("name, args, code", [
    ("tg_layernorm", but(NORM, a0=F64), N.TG_ERR_INVALID_ARGUMENT), ("tg_layernorm", but(NORM, a0=77), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_layernorm", but(NORM, a1=-1), N.TG_ERR_INVALID_ARGUMENT), ("tg_layernorm", but(NORM, a2=0), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_layernorm", but(NORM, a3=None), N.TG_ERR_INVALID_ARGUMENT), ("tg_layernorm", but(NORM, a12=None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_layernorm", but(NORM, a9=-1.0), N.TG_ERR_INVALID_ARGUMENT), ("tg_layernorm", but(NORM, a9=float("nan")), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_layernorm", but(NORM, a14=P), N.TG_ERR_INVALID_ARGUMENT), ("tg_layernorm", but(NORM, a4=7), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_layernorm", but(NORM, a5=P, a6=7), N.TG_ERR_DIMENSION_MISMATCH), ("tg_layernorm", but(NORM, a10=P, a11=7), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_layernorm", but(NORM, a13=7), N.TG_ERR_DIMENSION_MISMATCH), ("tg_layernorm", but(NORM, a2=1 << 31), N.TG_ERR_UNSUPPORTED),
    ("tg_layernorm_backward", but(NORM_BACK, a0=I32), N.TG_ERR_INVALID_ARGUMENT), ("tg_layernorm_backward", but(NORM_BACK, a3=None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_layernorm_backward", but(NORM_BACK, a10=None), N.TG_ERR_INVALID_ARGUMENT), ("tg_layernorm_backward", but(NORM_BACK, a4=7), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_layernorm_backward", but(NORM_BACK, a9=7), N.TG_ERR_DIMENSION_MISMATCH), ("tg_layernorm_backward", but(NORM_BACK, a13=7), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_layernorm_backward", but(NORM_BACK, a5=P, a6=7), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_blocks8_quantize", but(QUANT, a0=F64), N.TG_ERR_INVALID_ARGUMENT), ("tg_blocks8_quantize", but(QUANT, a2=-8), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_blocks8_quantize", but(QUANT, a3=None), N.TG_ERR_INVALID_ARGUMENT), ("tg_blocks8_quantize", but(QUANT, a5=None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_blocks8_quantize", but(QUANT, a7=None), N.TG_ERR_INVALID_ARGUMENT), ("tg_blocks8_quantize", but(QUANT, a10=P, a11=2), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_blocks8_quantize", but(QUANT, a4=7), N.TG_ERR_DIMENSION_MISMATCH), ("tg_blocks8_quantize", but(QUANT, a6=7), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_blocks8_quantize", but(QUANT, a10=P, a11=1, a12=P), N.TG_ERR_DIMENSION_MISMATCH), ("tg_blocks8_quantize", but(QUANT, a1=1 << 31), N.TG_ERR_UNSUPPORTED),
    ("tg_blocks8_quantize_tiles", but(TILES, a0=F64), N.TG_ERR_INVALID_ARGUMENT), ("tg_blocks8_quantize_tiles", but(TILES, a5=None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_blocks8_quantize_tiles", but(TILES, a10=P, a11=1), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_blocks8_transpose", (2, 8, None, 8, P, 2, None), N.TG_ERR_INVALID_ARGUMENT), ("tg_blocks8_transpose", (2, 8, P, 8, P, 1, None), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_blocks8_dequantize", but(VALUES, a3=64), N.TG_ERR_INVALID_ARGUMENT), ("tg_blocks8_dequantize", but(VALUES, a10=7), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_blocks8_layernorm", but(NORM8, a14=None), N.TG_ERR_INVALID_ARGUMENT), ("tg_blocks8_layernorm", but(NORM8, a13=7), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_blocks8_layernorm", but(NORM8, a12=None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_blocks8_gemm", but(GEMM, a0=F64), N.TG_ERR_INVALID_ARGUMENT), ("tg_blocks8_gemm", but(GEMM, a1=-4), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_blocks8_gemm", but(GEMM, a11=2), N.TG_ERR_INVALID_ARGUMENT), ("tg_blocks8_gemm", but(GEMM, a6=None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_blocks8_gemm", but(GEMM, a16=None), N.TG_ERR_INVALID_ARGUMENT), ("tg_blocks8_gemm", but(GEMM, a5=3), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_blocks8_gemm", but(GEMM, a10=3), N.TG_ERR_DIMENSION_MISMATCH), ("tg_blocks8_gemm", but(GEMM, a17=3), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_blocks8_gemm", but(GEMM, a1=1 << 31), N.TG_ERR_UNSUPPORTED), ("tg_blocks8_gemm", but(GEMM, a2=1 << 31, a17=1 << 31), N.TG_ERR_UNSUPPORTED),
    ("tg_token_logprobs", but(TOKENS, a0=F64), N.TG_ERR_INVALID_ARGUMENT), ("tg_token_logprobs", but(TOKENS, a2=0), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_token_logprobs", but(TOKENS, a10=33), N.TG_ERR_INVALID_ARGUMENT), ("tg_token_logprobs", but(TOKENS, a10=-1), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_token_logprobs", but(TOKENS, a10=9), N.TG_ERR_INVALID_ARGUMENT), ("tg_token_logprobs", but(TOKENS, a5=None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_token_logprobs", but(TOKENS, a11=None), N.TG_ERR_INVALID_ARGUMENT), ("tg_token_logprobs", but(TOKENS, a4=7), N.TG_ERR_DIMENSION_MISMATCH),
    ("tg_token_logprobs", but(TOKENS, a2=1 << 31, a4=1 << 31), N.TG_ERR_UNSUPPORTED),
    ("tg_token_logprobs_backward", but(TOKENS_BACK, a7=None), N.TG_ERR_INVALID_ARGUMENT), ("tg_token_logprobs_backward", but(TOKENS_BACK, a5=None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_token_logprobs_backward", but(TOKENS_BACK, a8=None), N.TG_ERR_INVALID_ARGUMENT), ("tg_token_logprobs_backward", but(TOKENS_BACK, a11=None), N.TG_ERR_INVALID_ARGUMENT),
    ("tg_token_logprobs_backward", but(TOKENS_BACK, a12=7), N.TG_ERR_DIMENSION_MISMATCH),
])
def test_abi_refusals(name, args, code):
    L = N.lib()
    assert getattr(L, name)(*args) == code
    assert len(L.tg_last_error()) > 0


def test_empty_problems_touch_nothing():
    L = N.lib()
    assert L.tg_layernorm(*but(NORM, a1=0, a3=None, a7=None, a8=None, a12=None)) == N.TG_OK
    assert L.tg_layernorm_backward(*but(NORM_BACK, a12=None, a14=None, a15=None)) == N.TG_OK
    assert L.tg_blocks8_quantize(*but(QUANT, a1=0, a3=None, a5=None, a7=None)) == N.TG_OK
    assert L.tg_blocks8_quantize_tiles(*but(TILES, a2=0, a3=None, a5=None, a7=None)) == N.TG_OK
    assert L.tg_blocks8_dequantize(*but(VALUES, a1=0, a4=None, a6=None, a9=None)) == N.TG_OK
    assert L.tg_blocks8_gemm(*but(GEMM, a1=0, a4=None, a6=None, a16=None)) == N.TG_OK
    assert L.tg_token_logprobs(*but(TOKENS, a1=0, a3=None, a5=None, a7=None)) == N.TG_OK
    assert L.tg_token_logprobs_backward(*but(TOKENS_BACK, a1=0, a3=None, a7=None, a11=None)) == N.TG_OK
