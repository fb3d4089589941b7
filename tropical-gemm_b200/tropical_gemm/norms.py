"""Layer norm, with the residual's addition, and its gradients.

    r = norms.layernorm(x, weight, bias, residual=x0)     # r.y the norm of r.h = x + x0

`tropical_gemm.pytorch.layernorm` is the same with autograd, and
`blocks8.layernorm` gives its output in 8-bit floating point.  The calls of this
module record no graph.

Tensors are CUDA tensors of float32, float16 or bfloat16 with any leading
dimensions; rows may be strided, their elements are contiguous (other layouts
are copied).  All calls run on torch's current stream and do not synchronise.
Wrong types, shapes and devices raise ValueError, CPU tensors RuntimeError,
and what the engine reports TropicalGemmError.
"""
from typing import NamedTuple, Optional, Tuple

import torch

from ._layers import ext as _x


class LayerNorm(NamedTuple):
    """What `layernorm` gives: the norm y, h = x + residual, and for the backward
    each row's mean and 1 / sqrt(variance + eps) (else None)."""
    y: torch.Tensor
    h: torch.Tensor
    mean: Optional[torch.Tensor]
    rstd: Optional[torch.Tensor]


def layernorm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
              residual: Optional[torch.Tensor] = None, eps: float = 1e-5, stats: bool = False) -> LayerNorm:
    """y = (h - mean) / sqrt(variance + eps) * weight + bias over the last
    dimension of h = x + residual.  Sums are float32, taken of the unrounded h.
    `weight` and `bias` are of x's type, or None (ones, zeros).  `stats` also
    keeps what `layernorm_backward` reads.  Without a residual h is x itself."""
    return LayerNorm(*_x().layernorm(x, weight, bias, residual, eps, stats))


def layernorm_backward(grad: torch.Tensor, h: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight: Optional[torch.Tensor] = None,
                       grad_h: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of `layernorm` with respect to x (and residual: the same),
    weight and bias, from the gradients of y and of h; all of h's type.  The
    sums over rows are float32 in a fixed order.

    With `residual`, `h` is the x that `layernorm` was given beside it, and their
    sum is formed in float32 as there.  The h that `layernorm` gives is that sum
    rounded to its type; taken in its place, a 16-bit one puts an error of half a
    step of h, over the row's spread, into (h - mean) rstd.  A float32 h is the
    sum itself and needs no parts."""
    return _x().layernorm_backward(grad, h, mean, rstd, weight, grad_h, residual)


__all__ = ["LayerNorm", "layernorm", "layernorm_backward"]
