"""Matrices held in 8-bit floating point with a scale for each block of 128.

A matrix in 8-bit blocks is `Blocks8(q, scale)`: q float8_e4m3fn (.., K), scale
float32.  `scale` has one value for each row and block of 128 columns
(.., ceil(K / 128)), which is what activations take, or, for a two-dimensional
matrix, one for each tile of 128 x 128 (ceil(N / 128), ceil(K / 128)), which is
what weights take: a matrix in tiles is in tiles transposed, too.

    w8 = blocks8.quantize_tiles(weight)                          # (N, K), once
    z = blocks8.matmul(blocks8.quantize(x), w8, dtype=x.dtype)    # tokens x output channels
    n = blocks8.layernorm(x, w, b, residual=r)                    # n.blocks goes to matmul, n.h = x + r

`tropical_gemm.pytorch.linear_blocks8` is the linear layer with autograd.  The
calls of this module record no graph.

The quantising calls take powers of two as scales, the least that brings a
block's largest magnitude to 448 or below, and round to nearest even, so that a
code is one rounding of its value.  A block that holds a NaN or an infinity has
scale NaN: what is made of it is NaN.  The products take any float32 scales
(the product of two that meet within float32's range).  Where all are powers of
two, which is found out on the device, those of many tokens are about twice as
fast with b in tiles, four times with b in rows.

Tensors are CUDA tensors (inputs float32, float16 or bfloat16) with any leading
dimensions; rows may be strided, their elements are contiguous (other layouts
are copied).  All calls run on torch's current stream and do not synchronise.
Wrong types, shapes and devices raise ValueError, CPU tensors RuntimeError,
and what the engine reports TropicalGemmError.
"""
from typing import NamedTuple, Optional, Tuple

import torch

from ._layers import ext as _x


class Blocks8(NamedTuple):
    """Codes (.., K) float8_e4m3fn and their scales (see the module)."""
    q: torch.Tensor
    scale: torch.Tensor


class NormBlocks8(NamedTuple):
    """What `layernorm` gives: the norm in 8-bit blocks, and h = x + residual."""
    blocks: Blocks8
    h: torch.Tensor


def quantize(x: torch.Tensor) -> Blocks8:
    """`x` with a scale for each row and block of 128 columns.  Rows of q lie a
    multiple of 16 bytes apart, which the products read without a copy."""
    return Blocks8(*_x().quantize(x))


def quantize_both(x: torch.Tensor) -> Tuple[Blocks8, Blocks8]:
    """`x` (.., K) in blocks along its rows, and x^T (K, tokens) in blocks along
    the tokens, from one read: the operands of a product and of its weight's gradient."""
    q, scale, qt, scale_t = _x().quantize_both(x)
    return Blocks8(q, scale), Blocks8(qt, scale_t)


def quantize_tiles(w: torch.Tensor) -> Blocks8:
    """`w` (N, K) with a scale for each tile of 128 x 128."""
    q, scale, _ = _x().quantize_tiles(w, False)
    return Blocks8(q, scale)


def transpose(w: Blocks8) -> Blocks8:
    """A matrix in tiles of 128 x 128, transposed (the same values)."""
    q, scale = w
    if q.dim() != 2 or tuple(scale.shape) != (-(-q.size(0) // 128), -(-q.size(1) // 128)):
        raise ValueError(f"transpose needs one scale per tile of 128 x 128: q is {tuple(q.shape)}, scale is {tuple(scale.shape)}")
    return Blocks8(_x().transpose(q), scale.detach().t())


def dequantize(b: Blocks8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that 8-bit blocks stand for: q * scale in float32, rounded to `dtype`."""
    q, scale = b
    return _x().dequantize(q, scale, dtype)


def layernorm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
              residual: Optional[torch.Tensor] = None, eps: float = 1e-5) -> NormBlocks8:
    """`norms.layernorm` with its output in 8-bit blocks along the rows, quantised
    from the unrounded float32 values."""
    q, scale, h = _x().layernorm_blocks8(x, weight, bias, residual, eps)
    return NormBlocks8(Blocks8(q, scale), h)


def matmul(a: Blocks8, b: Blocks8, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """A B^T + bias in `dtype`: a (.., K) tokens in blocks along their rows, b (N, K)
    output channels in blocks along their rows or in tiles, bias (N,) of type
    `dtype`.  Sums are float32; their order depends on the sizes (a token's bits may
    depend on how many tokens share the call), not on the run."""
    aq, a_scale = a
    bq, b_scale = b
    return _x().matmul(aq, a_scale, bq, b_scale, bias, dtype)


__all__ = ["Blocks8", "NormBlocks8", "quantize", "quantize_both", "quantize_tiles", "transpose", "dequantize", "layernorm", "matmul"]
