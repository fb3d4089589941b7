"""Plain 64-bit forms of layer norm, 8-bit block products and token log probabilities, and their tolerances."""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step, relative
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}   # where relative steps end
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def norm(x, residual=None, weight=None, bias=None, eps=1e-5):
    h = x.double() if residual is None else x.double() + residual.double()
    mean = h.mean(-1, keepdim=True)
    rstd = ((h - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    u = (h - mean) * rstd
    y = u if weight is None else u * weight.double()
    return h, u, rstd, y if bias is None else y + bias.double()


def norm_backward(g, u, rstd, weight=None, grad_h=None):
    g = g.double()
    a = g if weight is None else g * weight.double()
    gx = rstd * (a - a.mean(-1, keepdim=True) - u * (a * u).mean(-1, keepdim=True))
    k = u.shape[-1]
    return gx if grad_h is None else gx + grad_h.double(), (g * u).reshape(-1, k).sum(0), g.reshape(-1, k).sum(0)


def two_to(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e.to(torch.int32)) if not e.is_cuda else ((e.long() + 1023) << 52).view(torch.float64)


def steps(top):
    """The least power of two, from 2^-126 on, that brings top to 448 or below."""
    part, e = torch.frexp(top.double())
    e = torch.where(part > 0.875, e - 8, e - 9)
    return two_to(torch.where(top > 0, e, -126).clamp_min(-126))


def e4m3(v):
    """Nearest e4m3 value, ties to even, in 64 bits."""
    quantum = two_to(torch.frexp(v.abs().clamp_min(2.0 ** -6)).exponent - 4)
    return torch.round(v / quantum) * quantum


def blocks(x, tall=1):
    """(values in units of their scale, scales) of a matrix in blocks of tall x 128, 64 bits."""
    rows, cols = x.shape
    rb, cb = -(-rows // tall), -(-cols // 128)
    full = x.new_zeros(rb * tall, cb * 128, dtype=torch.float64)
    full[:rows, :cols] = x.double()
    step = steps(full.view(rb, tall, cb, 128).abs().amax((1, 3)))
    q = e4m3(full / step.repeat_interleave(tall, 0).repeat_interleave(128, 1))
    return q[:rows, :cols], step


def values(q, scale):
    """What codes and scales stand for, 64 bits."""
    rows, cols = q.shape
    s = scale.double()
    if s.shape[0] != rows:
        s = s.repeat_interleave(128, 0)[:rows]
    return q.double() * s.repeat_interleave(128, 1)[:, :cols]


def tokens(logits, ids, ignore=-100):
    """logprob, entropy, log p (rows, vocab) in 64 bits; a row of -infinity alone has logprob -infinity and entropy 0."""
    x = logits.double()
    empty = (x == -float("inf")).all(-1)
    logs = x - torch.logsumexp(x, -1, keepdim=True)
    logs = torch.where(empty[..., None], -float("inf"), logs)
    p = logs.exp()
    entropy = -torch.where(p > 0, p * logs, 0.0).sum(-1) if not torch.isnan(p).any() else -torch.where(p == 0, 0.0, p * logs).sum(-1)
    bad = (ids < 0) | (ids >= x.shape[-1])
    lp = logs.gather(-1, torch.where(bad, 0, ids)[..., None])[..., 0]
    lp = torch.where(bad, float("nan"), lp)
    return torch.where(ids == ignore, 0.0, lp), entropy, logs


def close(got, want, rel, floor=0.0):
    """|got - want| <= rel * |want| + floor, NaN and infinities where they are wanted."""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN elsewhere"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), "infinities elsewhere"
    limit = rel * want.abs() + floor
    off = torch.where(fine, (got - want).abs() - limit, -1.0)
    assert not (off > 0).any(), f"off by {float((got - want).abs()[off > 0].max())} at {int((off > 0).sum())} places, limit {float(limit[off > 0].min())}"
