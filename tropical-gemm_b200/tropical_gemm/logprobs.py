"""What a model answers with: log probabilities of tokens from rows of logits.

    r = logprobs.token_logprobs(logits, tokens, top=5)    # r.logprob, r.entropy, r.top_logprobs, r.top_tokens

`tropical_gemm.pytorch.token_logprobs` gives log probability and entropy with
autograd.  The calls of this module record no graph.

With p = softmax(row): logprob = log p[token], entropy = -sum p log p.  Logits of
-infinity (masked places) have no part in them.  A row of nothing else has
logprob and alternatives -infinity, entropy 0 and no gradient; a row that holds
a NaN or +infinity gives NaN.  `ignore_index` marks tokens that are none: their
logprob is 0 and passes no gradient.  Any other token outside the vocabulary
gives NaN.

Logits are CUDA tensors of float32, float16 or bfloat16 (.., vocabulary), tokens
int64 (..); rows may be strided, their elements are contiguous (other layouts
are copied).  All calls run on torch's current stream and do not synchronise.
Wrong types, shapes and devices raise ValueError, CPU tensors RuntimeError,
and what the engine reports TropicalGemmError.
"""
from typing import NamedTuple, Optional

import torch

from ._layers import ext as _x


class TokenLogprobs(NamedTuple):
    """What `token_logprobs` gives, float32: the tokens' log probabilities (None
    without tokens), the rows' entropies, the most likely tokens' log
    probabilities and these tokens (int64; None for top=0), and `stats` (.., 2),
    which the backward reads: the row's largest logit m and log sum exp(logit - m)."""
    logprob: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]
    stats: torch.Tensor


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of `tokens`, entropies, and the `top` (0 to 32) most likely
    tokens of each row from the most likely on; of equal logits the lower token
    comes first (as the tropical products take the lowest index)."""
    return TokenLogprobs(*_x().token_logprobs(logits, tokens, top, ignore_index))


def token_logprobs_backward(logits: torch.Tensor, tokens: Optional[torch.Tensor], stats: torch.Tensor, entropy: Optional[torch.Tensor] = None,
                            grad_logprob: Optional[torch.Tensor] = None, grad_entropy: Optional[torch.Tensor] = None,
                            ignore_index: int = -100) -> torch.Tensor:
    """Gradient of the logits from the gradients of logprob and entropy (float32,
    None for zeros) and what `token_logprobs` gave; of the logits' type."""
    return _x().token_logprobs_backward(logits, tokens, stats, entropy, grad_logprob, grad_entropy, ignore_index)


__all__ = ["TokenLogprobs", "token_logprobs", "token_logprobs_backward"]
