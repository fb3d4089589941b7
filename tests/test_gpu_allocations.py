"""What the 8-bit row calls and the layers allocate is seen by those who watch allocations: dispatch modes (memory trackers), and the
deterministic mode that fills memory which is not written."""
import contextlib

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import tropical_gemm.pytorch as tp
from tropical_gemm import blocks8, logprobs, norms, rows8

pytestmark = pytest.mark.gpu


class Allocated(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.bytes = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        r = func(*args, **(kwargs or {}))
        if func.overloadpacket in (torch.ops.aten.empty, torch.ops.aten.empty_strided, torch.ops.aten.empty_like):
            self.bytes += r.untyped_storage().nbytes()
        return r


def calls():
    x, w = torch.randn(6, 40, device="cuda"), torch.randn(24, 40, device="cuda")
    k, ids = torch.ones(40, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda")
    q, w8 = rows8.quantize(x), rows8.quantize(w)
    b, t8 = blocks8.quantize(x), blocks8.quantize_tiles(w)
    n = norms.layernorm(x, k, k, stats=True)
    leaf = x.clone().requires_grad_(True)
    return {
        "rows8.quantize": lambda: rows8.quantize(x), "rows8.dequantize": lambda: [rows8.dequantize(q)], "rows8.matmul": lambda: [rows8.matmul(q, w8)],
        "rmsnorm_linear_rows8": lambda: tp.rmsnorm_linear_rows8(leaf, k, w),
        "blocks8.quantize": lambda: blocks8.quantize(x), "blocks8.quantize_both": lambda: [s for b in blocks8.quantize_both(x) for s in b],
        "blocks8.quantize_tiles": lambda: blocks8.quantize_tiles(w), "blocks8.dequantize": lambda: [blocks8.dequantize(b)],
        "blocks8.matmul": lambda: [blocks8.matmul(b, t8)], "norms.layernorm": lambda: norms.layernorm(x, k, k, residual=x, stats=True),
        "norms.layernorm_backward": lambda: norms.layernorm_backward(x, x, n.mean, n.rstd, k),
        "logprobs.token_logprobs": lambda: logprobs.token_logprobs(x, ids, top=3), "linear_blocks8": lambda: [tp.linear_blocks8(leaf, w)],
    }


def tensors(out):
    return [t for t in (out if isinstance(out, (tuple, list)) else [out]) if isinstance(t, torch.Tensor)]


NAMES = ["rows8.quantize", "rows8.dequantize", "rows8.matmul", "rmsnorm_linear_rows8", "blocks8.quantize", "blocks8.quantize_both", "blocks8.quantize_tiles",
         "blocks8.dequantize", "blocks8.matmul", "norms.layernorm", "norms.layernorm_backward", "logprobs.token_logprobs", "linear_blocks8"]


@pytest.mark.parametrize("name", NAMES)
def test_dispatch_modes_see_outputs(name):
    call = calls()[name]
    want = [t.detach().clone() for t in tensors(call())]
    with Allocated() as seen:
        got = tensors(call())
    assert seen.bytes >= sum(t.untyped_storage().nbytes() for t in got) > 0
    for p, q in zip(got, want):
        assert torch.equal(p.detach().view(torch.uint8) if p.dtype == torch.float8_e4m3fn else p.detach(), q.view(torch.uint8) if q.dtype == torch.float8_e4m3fn else q)


@contextlib.contextmanager
def deterministic():
    before = torch.are_deterministic_algorithms_enabled(), torch.is_deterministic_algorithms_warn_only_enabled()
    torch.use_deterministic_algorithms(True)
    try:
        yield
    finally:
        torch.use_deterministic_algorithms(before[0], warn_only=before[1])


@pytest.mark.parametrize("name", NAMES)
def test_deterministic_mode(name):
    call = calls()[name]
    want = [t.detach().clone() for t in tensors(call())]
    with deterministic():
        got = tensors(call())
    for p, q in zip(got, want):
        assert torch.equal(p.detach().view(torch.uint8) if p.dtype == torch.float8_e4m3fn else p.detach(), q.view(torch.uint8) if q.dtype == torch.float8_e4m3fn else q)


def test_deterministic_mode_fills_what_is_not_written():
    x = torch.randn(6, 40, device="cuda")
    with deterministic():
        q = blocks8.quantize(x).q   # rows 48 bytes apart
        codes = torch.empty(0, dtype=torch.uint8, device="cuda").set_(q.untyped_storage())
        assert codes.numel() == 6 * 48 and (codes.view(6, 48)[:, 40:] & 0x7f == 0x7f).all()   # NaN
