"""Matrices held in 8-bit rows: the linear layers and norms beside a tropical layer.

A matrix in 8-bit rows is `Rows8(q, scale)`: row r stands for q[r] * scale[r],
q int8, scale f32.  One format serves the whole chain: the norm writes it, the
product reads it on the 8-bit tensor cores, and the backward reads the same
bytes again as the activations' checkpoint: a layer keeps two bytes per
element of x between its forward and its backward (the norm's output and h).

    r = rows8.rmsnorm(x, norm_weight, residual=x0)           # norm of x + x0, in 8 bits
    z = rows8.matmul(r.rows, rows8.quantize(weight))          # tokens x output channels

`tropical_gemm.pytorch.rmsnorm_linear_rows8` is the same chain with autograd.

Tensors are CUDA tensors of float32, float16 or bfloat16 with any leading
dimensions; rows may be strided, their elements are contiguous (other layouts
are copied).  All calls run on torch's current stream and do not synchronise.
"""
from typing import NamedTuple, Optional, Tuple

import torch

from . import _native as N

TYPES = {torch.float32: 0, torch.bfloat16: 4, torch.float16: 5}


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


def _type(t: torch.Tensor, what: str) -> int:
    code = TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    return code


def _on(dev: torch.device, *ts) -> None:
    if dev.type != "cuda":
        raise RuntimeError("the tropical-gemm engine needs CUDA tensors")
    for t in ts:
        if t is not None and t.device != dev:
            raise ValueError(f"Tensors must be on the same device: got {dev} and {t.device}")


def _flat(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """`t` as (rows, columns) and its row stride; a copy only where rows are
    not contiguous or cannot be flattened."""
    if t.is_contiguous():
        return t, t.size(-1)
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.reshape(_rows_of(t), t.shape[-1])
    t = N._rows(t)
    return t, N._ld(t)


def _rows_of(t: torch.Tensor) -> int:
    if t.dim() == 2:
        return t.size(0)
    n = 1
    for s in t.shape[:-1]:
        n *= s
    return n


def _check_rows8(r: Rows8, what: str) -> None:
    q, s = r
    if q.dtype != torch.int8 or s.dtype != torch.float32:
        raise ValueError(f"{what} must be int8 rows with float32 scales, got {q.dtype} and {s.dtype}")
    if q.dim() == 0 or s.shape != q.shape[:-1]:
        raise ValueError(f"{what} needs one scale per row: q is {tuple(q.shape)}, scale is {tuple(s.shape)}")


# the handle of torch's current stream, without the Stream object around it
# where this torch has that (2 us less per call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _call(dev: torch.device, fn, *args) -> None:
    i = dev.index
    if i == torch.cuda.current_device():
        status = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _raw_stream(i))
    if status:
        N.check(status)


def quantize(x: torch.Tensor) -> Rows8:
    """`x` in 8-bit rows: scale = max|row| / 127, q = x / scale rounded to
    nearest even.  A row of zeros (or below 2^-120) has scale 0; a row that
    holds a NaN or an infinity has scale NaN."""
    code = _type(x, "x")
    _on(x.device)
    if x.dim() == 0:
        raise ValueError("expected a tensor with at least one dimension")
    xf, ldx = _flat(x)
    shape = x.shape
    k = shape[-1]
    q = x.new_empty(shape, dtype=torch.int8)
    scale = x.new_empty(shape[:-1], dtype=torch.float32)
    _call(x.device, N.lib().tg_rows8_quantize, code, _rows_of(x), k, xf.data_ptr(), ldx, q.data_ptr(), k, scale.data_ptr())
    return Rows8(q, scale)


def dequantize(r: Rows8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that 8-bit rows stand for, rounded once to `dtype`."""
    _check_rows8(r, "rows")
    q, scale = r
    _on(q.device, scale)
    if dtype not in TYPES:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    qf, ldq = _flat(q)
    k = q.shape[-1]
    y = q.new_empty(q.shape, dtype=dtype)
    _call(q.device, N.lib().tg_rows8_dequantize, TYPES[dtype], _rows_of(q), k, qf.data_ptr(), ldq,
          scale.contiguous().data_ptr(), y.data_ptr(), k)
    return y


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
            checkpoint: bool = False) -> NormRows8:
    """Root-mean-square norm of h = x + residual over the last dimension,
    times `weight`, in 8-bit rows.  `checkpoint` also keeps h in 8-bit rows
    and the row's factor, which is what `rmsnorm_backward` reads.  Without a
    residual h is x itself."""
    code = _type(x, "x")
    dev = x.device
    _on(dev, weight, residual)
    shape = x.shape
    k = shape[-1] if shape else 0
    if k == 0:
        raise ValueError("x needs at least one column")
    if weight.dtype != x.dtype or weight.shape != (k,):
        raise ValueError(f"weight must be {x.dtype} of shape ({k},), got {weight.dtype} {tuple(weight.shape)}")
    if residual is not None and (residual.dtype != x.dtype or residual.shape != shape):
        raise ValueError(f"residual must be like x ({x.dtype} {tuple(x.shape)}), got {residual.dtype} {tuple(residual.shape)}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    rows, lead = _rows_of(x), shape[:-1]
    xf, ldx = _flat(x)
    weight = weight.contiguous()
    q = x.new_empty(shape, dtype=torch.int8)
    scale = x.new_empty(lead, dtype=torch.float32)
    rf, ldr, h, hp = None, 0, x, None
    if residual is not None:
        rf, ldr = _flat(residual)
        h = x.new_empty(shape)
        hp = h.data_ptr()
    ckpt = ckpt_scale = rstd = None
    if checkpoint:
        ckpt = x.new_empty(shape, dtype=torch.int8)
        ckpt_scale = x.new_empty(lead, dtype=torch.float32)
        rstd = x.new_empty(lead, dtype=torch.float32)
    _call(dev, N.lib().tg_rows8_rmsnorm, code, rows, k, xf.data_ptr(), ldx, None if rf is None else rf.data_ptr(), ldr,
          weight.data_ptr(), eps, hp, k, q.data_ptr(), k, scale.data_ptr(),
          None if ckpt is None else ckpt.data_ptr(), k, None if ckpt is None else ckpt_scale.data_ptr(),
          None if ckpt is None else rstd.data_ptr())
    return NormRows8(Rows8(q, scale), h, None if ckpt is None else Rows8(ckpt, ckpt_scale), rstd)


def rmsnorm_backward(grad: torch.Tensor, checkpoint: Rows8, rstd: torch.Tensor, weight: torch.Tensor,
                     grad_h: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of `rmsnorm` with respect to x (and residual: the same) and
    weight, from the gradients of its output and of h, and h's 8-bit
    checkpoint.  `grad` is float32 or of weight's type; the results are of
    weight's type.  The rounding to 8 bits passes gradients straight through."""
    _check_rows8(checkpoint, "checkpoint")
    ck, cs = checkpoint
    code, gcode = _type(weight, "weight"), _type(grad, "grad")
    dev = grad.device
    _on(dev, ck, cs, rstd, weight, grad_h)
    k = ck.shape[-1]
    if k == 0:
        raise ValueError("the checkpoint needs at least one column")
    if grad.shape != ck.shape:
        raise ValueError(f"grad must have the checkpoint's shape {tuple(ck.shape)}, got {tuple(grad.shape)}")
    if gcode != code and gcode != 0:
        raise ValueError(f"grad must be float32 or weight's {weight.dtype}, got {grad.dtype}")
    if weight.shape != (k,):
        raise ValueError(f"weight must have shape ({k},), got {tuple(weight.shape)}")
    if rstd.dtype != torch.float32 or rstd.shape != cs.shape:
        raise ValueError(f"rstd must be float32 of shape {tuple(cs.shape)}, got {rstd.dtype} {tuple(rstd.shape)}")
    if grad_h is not None and (grad_h.dtype != weight.dtype or grad_h.shape != grad.shape):
        raise ValueError(f"grad_h must be {weight.dtype} of shape {tuple(grad.shape)}, got {grad_h.dtype} {tuple(grad_h.shape)}")
    gf, ldg = _flat(grad)
    kf, ldk = _flat(ck)
    hf, ldh = (None, 0) if grad_h is None else _flat(grad_h)
    weight, cs, rstd = weight.contiguous(), cs.contiguous(), rstd.contiguous()
    grad_x = weight.new_empty(grad.shape)
    grad_w = weight.new_empty(k)
    _call(dev, N.lib().tg_rows8_rmsnorm_backward, code, gcode, _rows_of(ck), k, gf.data_ptr(), ldg,
          None if hf is None else hf.data_ptr(), ldh, weight.data_ptr(), kf.data_ptr(), ldk, cs.data_ptr(),
          rstd.data_ptr(), grad_x.data_ptr(), k, grad_w.data_ptr())
    return grad_x, grad_w


def matmul(a: Rows8, b: Rows8, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """A B^T + bias in `dtype`: a (.., K) tokens, b (N, K) output channels, both
    in 8-bit rows, bias (N,) of type `dtype`.  The integer sums are exact."""
    _check_rows8(a, "a")
    _check_rows8(b, "b")
    aq, asc = a
    bq, bsc = b
    dev = aq.device
    _on(dev, asc, bq, bsc, bias)
    if bq.dim() != 2:
        raise ValueError(f"b must be two-dimensional (channels, K), got {tuple(bq.shape)}")
    n, k = bq.shape
    if aq.shape[-1] != k:
        raise ValueError(f"Dimension mismatch: a has {aq.shape[-1]} columns, b has {k}")
    code = TYPES.get(dtype)
    if code is None:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    if bias is not None and (bias.dtype != dtype or bias.shape != (n,)):
        raise ValueError(f"bias must be {dtype} of shape ({n},), got {bias.dtype} {tuple(bias.shape)}")
    af, lda = _flat(aq)
    bf, ldb = _flat(bq)
    asc, bsc = asc.contiguous(), bsc.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    c = aq.new_empty(aq.shape[:-1] + (n,), dtype=dtype)
    _call(dev, N.lib().tg_rows8_gemm, code, _rows_of(aq), n, k, af.data_ptr(), lda, asc.data_ptr(), bf.data_ptr(), ldb,
          bsc.data_ptr(), None if bias is None else bias.data_ptr(), c.data_ptr(), n)
    return c


def matmul_backward(grad: torch.Tensor, a: Optional[Rows8], b: Optional[Rows8], dtype_a: Optional[torch.dtype] = None,
                    dtype_b: Optional[torch.dtype] = None) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients of `matmul` with respect to the values that `a` and `b` stand
    for: (grad B, grad^T A) in `dtype_a` and `dtype_b` (grad's type by
    default).  grad_A needs b only and grad_B needs a only; give None for the
    operand of a gradient that is not wanted.  Sums are float32; a bfloat16
    gradient meets the 8-bit values rounded once to bfloat16, float16 and
    float32 gradients are carried with 16 and 24 significant bits."""
    code = _type(grad, "grad")
    dev = grad.device
    _on(dev)
    if grad.dim() == 0:
        raise ValueError("expected a gradient with at least one dimension")
    n, rows = grad.shape[-1], _rows_of(grad)
    gf, ldg = _flat(grad)
    grad_a = grad_b = None
    for dt in (dtype_a, dtype_b):
        if dt is not None and dt not in TYPES:
            raise ValueError(f"gradients must be float32, float16 or bfloat16, got {dt}")
    if b is not None:
        _check_rows8(b, "b")
        _on(dev, *b)
        if b.q.dim() != 2 or b.q.shape[0] != n:
            raise ValueError(f"Dimension mismatch: grad is {tuple(grad.shape)}, b is {tuple(b.q.shape)}")
        k = b.q.shape[1]
        bf, ldb = _flat(b.q)
        scale = b.scale.contiguous()
        grad_a = grad.new_empty(grad.shape[:-1] + (k,), dtype=dtype_a or grad.dtype)
        _call(dev, N.lib().tg_rows8_gemm_backward, code, TYPES[grad_a.dtype], 0, rows, k, n, gf.data_ptr(), ldg,
              bf.data_ptr(), ldb, scale.data_ptr(), grad_a.data_ptr(), k)
    if a is not None:
        _check_rows8(a, "a")
        _on(dev, *a)
        if a.q.shape[:-1] != grad.shape[:-1]:
            raise ValueError(f"Dimension mismatch: grad is {tuple(grad.shape)}, a is {tuple(a.q.shape)}")
        k = a.q.shape[-1]
        af, lda = _flat(a.q)
        scale = a.scale.contiguous()
        grad_b = grad.new_empty((n, k), dtype=dtype_b or grad.dtype)
        _call(dev, N.lib().tg_rows8_gemm_backward, code, TYPES[grad_b.dtype], 1, n, k, rows, gf.data_ptr(), ldg,
              af.data_ptr(), lda, scale.data_ptr(), grad_b.data_ptr(), k)
    return grad_a, grad_b


def column_sum(x: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Sum over all but the last dimension (the gradient of `matmul`'s bias):
    float32 sums in a fixed order, in `dtype` (x's by default)."""
    code = _type(x, "x")
    _on(x.device)
    if dtype is not None and dtype not in TYPES:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    if x.dim() == 0:
        raise ValueError("expected a tensor with at least one dimension")
    xf, ldx = _flat(x)
    out = x.new_empty(x.shape[-1], dtype=dtype or x.dtype)
    _call(x.device, N.lib().tg_rows8_column_sum, code, TYPES[out.dtype], _rows_of(x), x.shape[-1], xf.data_ptr(), ldx,
          out.data_ptr())
    return out


__all__ = ["Rows8", "NormRows8", "quantize", "dequantize", "rmsnorm", "rmsnorm_backward", "matmul", "matmul_backward",
           "column_sum"]
