"""Products of 8-bit blocks whose scales are far from one and meet in the middle: what each scale does alone to a sum of codes (up to 2^24)
may pass f32's range, what both do does not.  Tolerances: test_gpu_blocks8.check_product."""
import pytest
import torch

import tropical_gemm.pytorch as tp
from tropical_gemm import blocks8
from tropical_gemm.blocks8 import Blocks8
from test_gpu_blocks8 import check_product

pytestmark = pytest.mark.gpu


# few tokens, one CTA for a sum and a cluster of them; pairs of CTAs, whole sums and split ones
@pytest.mark.parametrize("m, n, k", [(1, 130, 128), (3, 200, 300), (1, 256, 4096), (40, 130, 1000), (64, 512, 3000), (600, 600, 1000), (600, 600, 16384), (1100, 1300, 520)])
@pytest.mark.parametrize("ea, eb", [(118, -110), (-110, 118), (60, -60), (-118, 110), (110, -118)])
def test_scales_far_from_one(m, n, k, ea, eb):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    a = blocks8.quantize(torch.randn(m, k, generator=g, device="cuda"))
    w = torch.randn(n, k, generator=g, device="cuda")
    for b in (blocks8.quantize(w), blocks8.quantize_tiles(w)):
        for odd in (1.0, 1.3):   # powers of two, and others
            check_product(Blocks8(a.q, a.scale * (odd * 2.0 ** ea)), Blocks8(b.q, b.scale * 2.0 ** eb), torch.float32)


def test_values_far_from_one():
    """The same through the calls: activations of 1e-34, weights of 1e34."""
    for m in (1, 20, 700):
        x, w = torch.randn(m, 512, device="cuda") * 1e-34, torch.randn(384, 512, device="cuda") * 1e34
        a, b = blocks8.quantize(x), blocks8.quantize_tiles(w)
        check_product(a, b, torch.float32)
        assert torch.equal(tp.linear_blocks8(x, b), blocks8.matmul(a, b, dtype=torch.float32))
