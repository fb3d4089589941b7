"""A residual block with a tropical layer, its linear layers in 8-bit rows.

    h = x + r                     z = norm(h) W1^T           (8-bit rows)
    t = max_k(z[:, k] + T[k, :])                             (max-plus, argmax-scatter backward)
    y = h + norm(t) W2^T                                     (8-bit rows)

Trains the block on a synthetic target (activations kept in 8 bits between
forward and backward), then serves it with frozen 8-bit weights, all tokens at
once and one at a time.  Serving as many tokens as were trained on gives the
trained block's bits.  One token at a time gives them too at the sizes below;
wider norms of many tokens take their sums in another order than those of a
few, and a code next to a tie may come out as its neighbour.

    python examples/rows8_block.py [--steps 60] [--tokens 512] [--width 256]
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tropical-gemm_b200"))

import torch

from tropical_gemm import rows8
from tropical_gemm.pytorch import rmsnorm_linear_rows8, tropical_maxplus_matmul_gpu


class Block(torch.nn.Module):
    def __init__(self, width: int, inner: int):
        super().__init__()
        p = torch.nn.Parameter
        self.norm1, self.norm2 = p(torch.ones(width)), p(torch.ones(inner))
        self.w1 = p(torch.randn(inner, width) * width ** -0.5)
        self.tropical = p(torch.randn(inner, inner))
        self.w2 = p(torch.randn(width, inner) * inner ** -0.5)

    def forward(self, x, r):
        z, h = rmsnorm_linear_rows8(x, self.norm1, self.w1, residual=r)
        t = tropical_maxplus_matmul_gpu(z, self.tropical)
        y, _ = rmsnorm_linear_rows8(t, self.norm2, self.w2)
        return h + y

    @torch.no_grad()
    def frozen(self):
        """The weights in 8-bit rows, quantised once, and the serving path over them."""
        w1, w2 = rows8.quantize(self.w1), rows8.quantize(self.w2)

        @torch.no_grad()
        def serve(x, r):
            n = rows8.rmsnorm(x, self.norm1, residual=r)
            t = tropical_maxplus_matmul_gpu(rows8.matmul(n.rows, w1, dtype=x.dtype), self.tropical)
            return n.h + rows8.matmul(rows8.rmsnorm(t, self.norm2).rows, w2, dtype=x.dtype)

        return serve


def main(steps: int = 60, tokens: int = 512, width: int = 256, seed: int = 0):
    torch.manual_seed(seed)
    dev = torch.device("cuda", torch.cuda.current_device())
    block, teacher = Block(width, width // 2).to(dev), Block(width, width // 2).to(dev)
    x, r = torch.randn(tokens, width, device=dev), torch.randn(tokens, width, device=dev)
    with torch.no_grad():
        target = teacher(x, r)
    opt = torch.optim.Adam(block.parameters(), lr=1e-2)
    losses = []
    for _ in range(steps):
        opt.zero_grad(set_to_none=True)
        loss = (block(x, r) - target).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    serve = block.frozen()
    with torch.no_grad():
        trained = block(x, r)
    together = serve(x, r)
    single = torch.cat([serve(x[i:i + 1], r[i:i + 1]) for i in range(4)])
    return {"first": float(losses[0]), "last": float(losses[-1]),
            "served equals trained": bool(torch.equal(trained, together)),
            "one token at a time equals all": bool(torch.equal(single, together[:4]))}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--width", type=int, default=256)
    for k, v in main(**vars(ap.parse_args())).items():
        print(f"{k}: {v}")
