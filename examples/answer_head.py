"""The end of a language model behind a tropical layer: norm, vocabulary projection in 8-bit floating point, log probabilities.

    t = max_k(x[:, k] + T[k, :])                 (max-plus, argmax-scatter backward)
    y, h = layernorm(t + x)                      (residual, norm)
    logits = y W^T                               (e4m3 blocks of 128, tiles of 128 x 128)
    loss = -mean log p[token] - c * entropy      (no probabilities are stored)

Trains it on a synthetic rule, then serves it with the weight quantised once:
the norm's output goes to the product in 8 bits, and each row answers with its
most likely tokens.

    python examples/answer_head.py [--steps 40] [--rows 256] [--width 128] [--vocab 1000]
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tropical-gemm_b200"))

import torch

from tropical_gemm import blocks8, logprobs
from tropical_gemm.pytorch import layernorm, linear_blocks8, token_logprobs, tropical_maxplus_matmul_gpu


class Head(torch.nn.Module):
    def __init__(self, width: int, vocab: int):
        super().__init__()
        p = torch.nn.Parameter
        self.tropical = p(torch.randn(width, width))
        self.scale, self.shift = p(torch.ones(width)), p(torch.zeros(width))
        self.weight = p(torch.randn(vocab, width) * width ** -0.5)

    def forward(self, x):
        y, _ = layernorm(tropical_maxplus_matmul_gpu(x, self.tropical), self.scale, self.shift, residual=x)
        return linear_blocks8(y, self.weight)

    @torch.no_grad()
    def frozen(self):
        """The serving path over the weight in 8-bit tiles, quantised once."""
        w8 = blocks8.quantize_tiles(self.weight)

        @torch.no_grad()
        def serve(x, top):
            n = blocks8.layernorm(tropical_maxplus_matmul_gpu(x, self.tropical), self.scale, self.shift, residual=x)
            return logprobs.token_logprobs(blocks8.matmul(n.blocks, w8, dtype=x.dtype), top=top)

        return serve


def main(steps: int = 40, rows: int = 256, width: int = 128, vocab: int = 1000, entropy: float = 0.01, seed: int = 0):
    torch.manual_seed(seed)
    head = Head(width, vocab).to(torch.device("cuda", torch.cuda.current_device()))
    x = torch.randn(rows, width, device=head.weight.device)
    tokens = x.argmax(1) % vocab
    opt = torch.optim.Adam(head.parameters(), lr=1e-2)
    losses = []
    for _ in range(steps):
        opt.zero_grad(set_to_none=True)
        lp, h = token_logprobs(head(x), tokens)
        loss = -lp.mean() - entropy * h.mean()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    with torch.no_grad():
        trained = logprobs.token_logprobs(head(x), top=5)
    served = head.frozen()(x, 5)
    return {"first": float(losses[0]), "last": float(losses[-1]),
            "tokens answered": float((served.top_tokens[:, 0] == tokens).float().mean()),
            "answers as trained": float((served.top_tokens[:, 0] == trained.top_tokens[:, 0]).float().mean())}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("steps", 40), ("rows", 256), ("width", 128), ("vocab", 1000)):
        ap.add_argument(f"--{name}", type=int, default=value)
    for k, v in main(**vars(ap.parse_args())).items():
        print(f"{k}: {v}")
