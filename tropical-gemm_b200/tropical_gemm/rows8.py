"""Matrices held in 8-bit rows: the linear layers and norms beside a tropical layer.

A matrix in 8-bit rows is `Rows8(q, scale)`: row r stands for q[r] * scale[r],
q int8, scale f32.  One format serves the whole chain: the norm writes it, the
product reads it on the 8-bit tensor cores, and the backward reads the same
bytes again as the activations' checkpoint: a layer keeps two bytes per
element of x between its forward and its backward (the norm's output and h).

    r = rows8.rmsnorm(x, norm_weight, residual=x0)           # norm of x + x0, in 8 bits
    z = rows8.matmul(r.rows, rows8.quantize(weight))          # tokens x output channels

`tropical_gemm.pytorch.rmsnorm_linear_rows8` is the same chain with autograd.
The calls of this module record no graph: what they return requires no
gradient, whatever their arguments do, and `rmsnorm_backward`, `matmul_backward`
and `column_sum` are how gradients are taken.  (Without a residual `rmsnorm`
hands x through as h, as it came.)

Tensors are CUDA tensors of float32, float16 or bfloat16 with any leading
dimensions; rows may be strided, their elements are contiguous (other layouts
are copied).  All calls run on torch's current stream and do not synchronise.
Wrong types, shapes and devices raise ValueError, CPU tensors RuntimeError,
and what the engine reports TropicalGemmError.
"""
import os
from typing import NamedTuple, Optional, Tuple

import torch

from . import _native as N

_ext = None


def _x():
    """The torch binding (raises if it has not been built)."""
    global _ext
    if _ext is None:
        N.lib()
        path = os.path.join(os.path.dirname(N.LIB_PATH), "_rows8_torch.so")
        if not os.path.exists(path):
            raise ImportError(f"{path} not found: build it with `python __graft_entry__.py build` "
                              "(or `make -C tropical-gemm_b200 torch`)")
        from . import _rows8_torch
        _ext = _rows8_torch
    return _ext


class Rows8(NamedTuple):
    """(.., K) values q * scale[.., None]: q int8 (.., K), scale float32 (..)."""
    q: torch.Tensor
    scale: torch.Tensor


class NormRows8(NamedTuple):
    """What `rmsnorm` gives: the norm in 8-bit rows, h = x + residual, and for
    the backward h in 8-bit rows and 1 / sqrt(mean(h^2) + eps) (else None)."""
    rows: Rows8
    h: torch.Tensor
    checkpoint: Optional[Rows8]
    rstd: Optional[torch.Tensor]


def quantize(x: torch.Tensor) -> Rows8:
    """`x` in 8-bit rows: scale = max|row| / 127, q = x / scale rounded to
    nearest even.  A row of zeros (or below 2^-120) has scale 0; a row that
    holds a NaN or an infinity has scale NaN."""
    return Rows8(*_x().quantize(x))


def dequantize(r: Rows8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that 8-bit rows stand for: q * scale in float32, rounded to `dtype`."""
    q, scale = r
    return _x().dequantize(q, scale, dtype)


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
            checkpoint: bool = False) -> NormRows8:
    """Root-mean-square norm of h = x + residual over the last dimension,
    times `weight`, in 8-bit rows.  `checkpoint` also keeps h in 8-bit rows
    and the row's factor, which is what `rmsnorm_backward` reads.  Without a
    residual h is x itself.  The order of a row's sum of squares may depend on
    the number of rows; h and the checkpoint do not."""
    q, scale, h, ck, ck_scale, rstd = _x().rmsnorm(x, weight, residual, eps, checkpoint)
    return NormRows8(Rows8(q, scale), h, None if ck is None else Rows8(ck, ck_scale), rstd)


def rmsnorm_backward(grad: torch.Tensor, checkpoint: Rows8, rstd: torch.Tensor, weight: torch.Tensor,
                     grad_h: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of `rmsnorm` with respect to x (and residual: the same) and
    weight, from the gradients of its output and of h, and h's 8-bit
    checkpoint.  `grad` is float32 or of weight's type; the results are of
    weight's type.  The rounding to 8 bits passes gradients straight through."""
    q, scale = checkpoint
    return _x().rmsnorm_backward(grad, q, scale, rstd, weight, grad_h)


def matmul(a: Rows8, b: Rows8, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """A B^T + bias in `dtype`: a (.., K) tokens, b (N, K) output channels, both
    in 8-bit rows, bias (N,) of type `dtype`.  The integer sums are exact;
    K is below 131072."""
    aq, a_scale = a
    bq, b_scale = b
    return _x().matmul(aq, a_scale, bq, b_scale, bias, dtype)


def matmul_backward(grad: torch.Tensor, a: Optional[Rows8], b: Optional[Rows8], dtype_a: Optional[torch.dtype] = None,
                    dtype_b: Optional[torch.dtype] = None) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients of `matmul` with respect to the values that `a` and `b` stand
    for: (grad B, grad^T A) in `dtype_a` and `dtype_b` (grad's type by
    default).  grad_A needs b only and grad_B needs a only; give None for the
    operand of a gradient that is not wanted.  Sums are float32; a bfloat16
    gradient meets the 8-bit values rounded once to bfloat16, float16 and
    float32 gradients are carried with 16 and 24 significant bits."""
    aq, a_scale = a if a is not None else (None, None)
    bq, b_scale = b if b is not None else (None, None)
    return _x().matmul_backward(grad, aq, a_scale, bq, b_scale, dtype_a, dtype_b)


def column_sum(x: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Sum over all but the last dimension (the gradient of `matmul`'s bias):
    float32 sums in a fixed order, in `dtype` (x's by default)."""
    return _x().column_sum(x, dtype)


__all__ = ["Rows8", "NormRows8", "quantize", "dequantize", "rmsnorm", "rmsnorm_backward", "matmul", "matmul_backward",
           "column_sum"]
