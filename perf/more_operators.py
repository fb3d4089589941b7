"""The end of a language model at the sizes it is used at: layer norm, linear layers in 8-bit floating point, log probabilities of tokens.

Cases, their plain forms, and their definition in 64 bits.

    norm      h = x + residual, y = (h - mean) / sqrt(var + eps) * weight + bias over each row
    normstep  the same with its gradients, as a training step calls it
    linear    z = x W^T + bias; x held in e4m3 with a scale for each row's block of 128, W for each tile of 128 x 128
    normlin   norm and linear as a decoder calls them
    linstep   the linear with its gradients: grad W and grad^T x, the gradient too in e4m3 blocks along each sum
    tokens    log probabilities of given tokens, the rows' entropies, and the most likely alternatives
    tokstep   the first two with the gradient of the logits, as a training step calls them

A block's scale is the least power of two that brings its largest magnitude to 448 or below; codes are rounded to nearest even.

`own` False: elementary torch operations in 32 bits.  `own` True: the calls a user makes of the framework.
"""
import os
import sys

import torch

own = False

EPS = 1e-5
BLOCK = 128
IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a decoder: latency
        {"name": "norm one token", "op": "norm", "rows": 1, "cols": 4096, "type": "bf16", "residual": True},
        # a ragged batch of prompts of odd width, no residual
        {"name": "norm odd f16", "op": "norm", "rows": 777, "cols": 5001, "type": "f16", "residual": False},
        # a small f32 model's training step
        {"name": "norm step ragged f32", "op": "normstep", "rows": 1777, "cols": 1111, "type": "f32"},
        # a training batch
        {"name": "norm step training batch", "op": "normstep", "rows": 8192, "cols": 8192, "type": "bf16"},
        # one token through a projection: the weights' read
        {"name": "linear one token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": False},
        # a short prompt of odd length, odd widths, with a bias
        {"name": "linear odd", "op": "linear", "m": 333, "n": 1531, "k": 1111, "type": "f32", "bias": True},
        # a long prompt through a wide projection
        {"name": "linear prompt", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "bias": False},
        # sixteen sequences decoding together
        {"name": "norm and linear, sixteen", "op": "normlin", "m": 16, "n": 8192, "k": 4096, "type": "bf16"},
        # a training step of a layer
        {"name": "linear step", "op": "linstep", "m": 4096, "n": 4096, "k": 4096, "type": "bf16"},
        # one token's answer over a large vocabulary, with alternatives
        {"name": "tokens one answer", "op": "tokens", "rows": 1, "vocab": 131072, "top": 20, "type": "bf16"},
        # a prompt scored over a vocabulary of odd size
        {"name": "tokens prompt", "op": "tokens", "rows": 1531, "vocab": 50001, "top": 5, "type": "f16"},
        # the loss of a training batch and its gradient
        {"name": "tokens step", "op": "tokstep", "rows": 4096, "vocab": 65536, "type": "bf16"},
    ]


def draw(rng):
    def size(lo, hi):
        v = int(round(lo * (hi / lo) ** rng.random()))
        return v // 32 * 32 if rng.random() < 0.5 and v >= 64 else v

    op = rng.choice(["norm", "normstep", "linear", "linear", "normlin", "linstep", "tokens", "tokens", "tokstep"])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("norm", "normstep"):
        case = {"op": op, "rows": size(1, 8192), "cols": size(64, 8192), "type": t}
        if op == "norm":
            case["residual"] = rng.random() < 0.5
    elif op == "linear":
        case = {"op": op, "m": size(1, 8192), "n": size(64, 8192), "k": size(64, 8192), "type": t, "bias": rng.random() < 0.3}
    elif op == "normlin":
        case = {"op": op, "m": size(1, 256), "n": size(64, 8192), "k": size(64, 8192), "type": rng.choice(["bf16", "f16"])}
    elif op == "linstep":
        case = {"op": op, "m": size(1, 4096), "n": size(64, 4096), "k": size(64, 4096), "type": t}
    else:
        vocab = size(64, 131072)
        case = {"op": op, "rows": size(1, min(4096, 2 ** 28 // vocab)), "vocab": vocab, "type": t}
        if op == "tokens":
            case["top"] = rng.choice([0, 1, rng.randint(1, 32), rng.randint(1, 32)])
    return case


def work(case):
    e, op = BYTES[case["type"]], case["op"]
    if op in ("norm", "normstep"):
        n, c = case["rows"] * case["cols"], case["cols"]
        if op == "norm":  # x, y; with a residual it and h
            return {"bytes": e * (n * (4 if case["residual"] else 2) + 2 * c), "flops": 8 * n}
        return {"bytes": e * (7 * n + 4 * c), "flops": 20 * n}  # x, residual, y, h; gradients of y, h and x
    if op in ("tokens", "tokstep"):
        n, r = case["rows"] * case["vocab"], case["rows"]
        if op == "tokens":
            return {"bytes": e * n + r * (16 + 12 * case["top"]), "flops": 5 * n}
        return {"bytes": 2 * e * n + 24 * r, "flops": 12 * n}  # logits, their gradient
    m, n, k = case["m"], case["n"], case["k"]
    if op == "linear":  # x, the weights' codes, z
        return {"bytes": e * m * (k + n) + n * k, "flops": 2 * m * n * k}
    if op == "normlin":
        return {"bytes": e * m * (3 * k + n) + n * k, "flops": 2 * m * n * k}
    return {"bytes": 2 * e * (m * k + n * k + m * n), "flops": 6 * m * n * k}  # x, weight, z and their gradients


# --------------------------------------------------------------------------------------------------------------- inputs
def _step_of(top):  # 2^e with top / 2^e <= 448 = 0.875 * 2^9, e least and not below -126
    part, e = torch.frexp(top)
    e = torch.where(part > 0.875, e - 8, e - 9)
    e = torch.where(top > 0, e, -126).clamp_min(-126)
    return ((e + 127) << 23).view(torch.float32)  # its bits: a power taken by pow() may be off in the last place


def _rows8(x):
    """x (rows, cols) f32 as codes and one scale for each row's block of 128."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols)).view(rows, blocks, BLOCK)
    step = _step_of(v.abs().amax(2))
    return (v / step[:, :, None]).to(torch.float8_e4m3fn).view(rows, -1)[:, :cols], step


def _tiles8(w):
    """w (rows, cols) f32 as codes and one scale for each tile of 128 x 128."""
    rows, cols = w.shape
    rb, cb = -(-rows // BLOCK), -(-cols // BLOCK)
    v = torch.nn.functional.pad(w, (0, cb * BLOCK - cols, 0, rb * BLOCK - rows)).view(rb, BLOCK, cb, BLOCK)
    step = _step_of(v.abs().amax((1, 3)))
    q = (v / step[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(rb * BLOCK, cb * BLOCK)[:rows, :cols], step  # rows keep their pitch, a multiple of 128 bytes


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def hidden(rows, cols):  # hidden states: a few channels are much larger than the others, and no channel has mean zero
        return normal(rows, cols) * torch.where(uniform(cols) < 0.01, 8.0, 1.0) + 0.5 * normal(cols)

    op = case["op"]
    s = {"case": dict(case)}
    if op in ("norm", "normstep", "normlin"):
        r, c = (case["m"], case["k"]) if op == "normlin" else (case["rows"], case["cols"])
        s["x"] = normal(r, c).to(t) if op != "norm" or case["residual"] else hidden(r, c).to(t)
        s["x"][3::97] = 0  # padding tokens
        s["residual"] = hidden(r, c).to(t) if op != "norm" or case["residual"] else None
        if s["residual"] is not None:
            s["residual"][3::97] = 0
        s["weight"], s["bias"] = (1 + 0.2 * normal(c)).to(t), (0.2 * normal(c)).to(t)
        if op == "normstep":
            s["grad"], s["grad_h"] = normal(r, c).to(t), normal(r, c).to(t)
            for name in ("x", "residual", "weight", "bias"):
                s[name].requires_grad_(True)
        if op == "normlin":
            s["q"], s["scale"] = _tiles8(normal(case["n"], c) * c ** -0.5)
    elif op in ("linear", "linstep"):
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = hidden(m, k).to(t)
        w = normal(n, k) * k ** -0.5
        s["bias"] = normal(n).to(t) if op == "linstep" or case["bias"] else None
        if op == "linear":
            s["q"], s["scale"] = _tiles8(w)
        else:
            s["w"], s["grad"] = w.to(t), (normal(m, n) * 10 ** (2 * uniform(m, 1) - 3)).to(t)  # tokens weigh differently in a loss
            for name in ("x", "w", "bias"):
                s[name].requires_grad_(True)
    else:
        r, v = case["rows"], case["vocab"]
        logits = normal(r, v) * (1 + 2 * uniform(r, 1)) + 2 * normal(v)  # some rows are surer than others, some tokens commoner
        logits[:, v - v // 64:] = -float("inf")  # places of the vocabulary that hold no token
        s["logits"] = logits.to(t)
        s["tokens"] = torch.randint(0, v - v // 64, (r,), generator=g, device="cuda")
        if op == "tokstep":
            s["tokens"][uniform(r) < 0.03] = IGNORE  # padding
            s["grad"], s["grad_entropy"] = -uniform(r) / r, 0.1 * normal(r) / r
            s["logits"].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------ plain form
def _norm(x, residual, weight, bias):
    h = x.float() if residual is None else x.float() + residual.float()
    off = h - h.mean(1, keepdim=True)
    unit = off * torch.rsqrt(off.square().mean(1, keepdim=True) + EPS)
    return h, unit, unit * weight.float() + bias.float()


def _rows_values(q, step):
    return q.float() * step.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _tiles_values(q, step):
    return q.float() * step.repeat_interleave(BLOCK, 0)[:q.shape[0]].repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _plain(s):
    case = s["case"]
    op, t = case["op"], TYPES[case["type"]]
    if op == "norm":
        h, _, y = _norm(s["x"], s["residual"], s["weight"], s["bias"])
        return [y.to(t)] if s["residual"] is None else [y.to(t), h.to(t)]
    if op == "normstep":
        with torch.no_grad():
            h, unit, y = _norm(s["x"], s["residual"], s["weight"], s["bias"])
            off = h - h.mean(1, keepdim=True)
            rstd = torch.rsqrt(off.square().mean(1, keepdim=True) + EPS)
            g = s["grad"].float()
            inner = g * s["weight"].float()
            grad_x = rstd * (inner - inner.mean(1, keepdim=True) - unit * (inner * unit).mean(1, keepdim=True)) + s["grad_h"].float()
            return [y.to(t), h.to(t), grad_x.to(t), (g * unit).sum(0).to(t), g.sum(0).to(t)]
    if op == "normlin":
        h, _, y = _norm(s["x"], s["residual"], s["weight"], s["bias"])
        return [(_rows_values(*_rows8(y)) @ _tiles_values(s["q"], s["scale"]).t()).to(t), h.to(t)]
    if op == "linear":
        z = _rows_values(*_rows8(s["x"].float())) @ _tiles_values(s["q"], s["scale"]).t()
        return (z if s["bias"] is None else z + s["bias"].float()).to(t)
    if op == "linstep":
        with torch.no_grad():
            x, w, g = s["x"].float(), _tiles_values(*_tiles8(s["w"].float())), s["grad"].float()
            z = _rows_values(*_rows8(x)) @ w.t() + s["bias"].float()
            grad_w = _rows_values(*_rows8(g.t().contiguous())) @ _rows_values(*_rows8(x.t().contiguous())).t()
            return [z.to(t), (_rows_values(*_rows8(g)) @ w).to(t), grad_w.to(t), g.sum(0).to(t)]
    with torch.no_grad():
        raw = s["logits"].float()
        x = raw - raw.amax(1, keepdim=True)
        e = torch.exp(x)
        total = e.sum(1, keepdim=True)
        p, logs = e / total, x - torch.log(total)
        entropy = -torch.where(p > 0, p * logs, 0.0).sum(1)
        kept = s["tokens"] != IGNORE
        at = torch.where(kept, s["tokens"], 0)[:, None]
        logprob = torch.where(kept, logs.gather(1, at)[:, 0], 0.0)
        if op == "tokstep":
            grad = torch.where(kept, s["grad"], 0.0)[:, None]
            grad_x = -p * grad - torch.where(p > 0, p * (logs + entropy[:, None]), 0.0) * s["grad_entropy"][:, None]
            grad_x.scatter_add_(1, at, grad)
            return [logprob, entropy, grad_x.to(t)]
        if case["top"] == 0:
            return [logprob, entropy]
        # one whole number for each place, larger for larger values, and of equal values for the lower place
        place = torch.arange(x.shape[1], device=x.device)
        bits = (raw + 0.0).view(torch.int32).long()  # one zero, not two
        order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * 2 ** 20 + (2 ** 20 - 1 - place)
        ids = torch.topk(order, case["top"], 1).indices
        return [logprob, entropy, logs.gather(1, ids), ids]


# --------------------------------------------------------------------------------------------------- the framework's calls
def _package():
    if "tropical_gemm" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "tropical-gemm_b200"))
    import tropical_gemm.blocks8
    import tropical_gemm.logprobs
    import tropical_gemm.norms
    import tropical_gemm.pytorch
    return tropical_gemm


def _own(s):
    tg = _package()
    case = s["case"]
    op, t = case["op"], TYPES[case["type"]]
    if op == "norm":
        r = tg.norms.layernorm(s["x"], s["weight"], s["bias"], residual=s["residual"], eps=EPS)
        return [r.y] if s["residual"] is None else [r.y, r.h]
    if op == "normstep":
        y, h = tg.pytorch.layernorm(s["x"], s["weight"], s["bias"], residual=s["residual"], eps=EPS)
        grad_x, _, grad_w, grad_b = torch.autograd.grad((y, h), (s["x"], s["residual"], s["weight"], s["bias"]), (s["grad"], s["grad_h"]))
        return [y, h, grad_x, grad_w, grad_b]
    if op == "normlin":
        r = tg.blocks8.layernorm(s["x"], s["weight"], s["bias"], residual=s["residual"], eps=EPS)
        return [tg.blocks8.matmul(r.blocks, tg.blocks8.Blocks8(s["q"], s["scale"]), dtype=t), r.h]
    if op == "linear":
        return tg.blocks8.matmul(tg.blocks8.quantize(s["x"]), tg.blocks8.Blocks8(s["q"], s["scale"]), bias=s["bias"], dtype=t)
    if op == "linstep":
        z = tg.pytorch.linear_blocks8(s["x"], s["w"], s["bias"])
        return [z, *torch.autograd.grad(z, (s["x"], s["w"], s["bias"]), s["grad"])]
    if op == "tokstep":
        logprob, entropy = tg.pytorch.token_logprobs(s["logits"], s["tokens"], ignore_index=IGNORE)
        return [logprob, entropy, *torch.autograd.grad((logprob, entropy), s["logits"], (s["grad"], s["grad_entropy"]))]
    r = tg.logprobs.token_logprobs(s["logits"], s["tokens"], top=case["top"], ignore_index=IGNORE)
    return [r.logprob, r.entropy, r.top_logprobs, r.top_tokens] if case["top"] else [r.logprob, r.entropy]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    s = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    op = case["op"]

    def two_to(e):  # exactly
        return ((e.long() + 1023) << 52).view(torch.float64)

    def held(v, tall):  # the values that blocks of tall x 128 stand for
        rows, cols = v.shape
        full = v.new_zeros(-(-rows // tall) * tall, -(-cols // BLOCK) * BLOCK)
        full[:rows, :cols] = v
        b = full.unflatten(1, (-1, BLOCK)).unflatten(0, (-1, tall)).abs()
        top = b.amax(dim=(1, 3)).clamp_min(2.0 ** -200)
        tries = torch.floor(torch.log2(top)) - 9 + torch.arange(4, device=v.device, dtype=v.dtype)[:, None, None]
        e = tries.masked_fill(top * two_to(-tries) > 448, 900).amin(0)
        step = two_to(e.clamp_min(-126)).repeat_interleave(tall, 0).repeat_interleave(BLOCK, 1)
        y = full / step
        size = y.abs().clamp_min(2.0 ** -6)
        quantum = two_to(torch.frexp(size).exponent - 4)
        return (torch.round(y / quantum) * quantum * step)[:rows, :cols]

    def norm(x, residual):
        h = x if residual is None else x + residual
        mean = h.sum(1, keepdim=True) / h.shape[1]
        rstd = ((h - mean).pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).pow(-0.5)
        return h, rstd, (h - mean) * rstd

    if op in ("norm", "normstep", "normlin"):
        h, rstd, u = norm(s["x"], s["residual"])
        y = u * s["weight"] + s["bias"]
        if op == "norm":
            return [y] if s["residual"] is None else [y, h]
        if op == "normlin":
            return [torch.mm(held(y, 1), (s["q"].double() * s["scale"].repeat_interleave(BLOCK, 0)[:case["n"]].repeat_interleave(BLOCK, 1)[:, :case["k"]]).T), h]
        a = s["grad"] * s["weight"]
        k = h.shape[1]
        grad_x = rstd * (a - a.sum(1, keepdim=True) / k - u * torch.einsum("ij,ij->i", a, u)[:, None] / k)
        return [y, h, grad_x + s["grad_h"], torch.einsum("ij,ij->j", s["grad"], u), torch.einsum("ij->j", s["grad"])]
    if op == "linear":
        w = s["q"].double() * s["scale"].repeat_interleave(BLOCK, 0)[:case["n"]].repeat_interleave(BLOCK, 1)[:, :case["k"]]
        z = torch.mm(held(s["x"], 1), w.T)
        return z if s["bias"] is None else z + s["bias"][None]
    if op == "linstep":
        w = held(s["w"], BLOCK)
        grad_w = torch.mm(held(s["grad"].T.contiguous(), 1), held(s["x"].T.contiguous(), 1).T)
        return [torch.addmm(s["bias"], held(s["x"], 1), w.T), torch.mm(held(s["grad"], 1), w), grad_w, torch.einsum("ij->j", s["grad"])]
    logits = s["logits"]
    logs = logits - torch.logsumexp(logits, 1, keepdim=True)
    p = logs.exp()
    finite = logs.clamp_min(-1e4)  # where p is zero its product is zero
    entropy = -torch.einsum("ij,ij->i", p, finite)
    rows = torch.arange(logits.shape[0], device=logits.device)
    kept = (s["tokens"] >= 0).double()
    at = s["tokens"].clamp_min(0)
    logprob = logs[rows, at] * kept
    if op == "tokstep":
        a = (s["grad"] * kept)[:, None]
        grad = -a * p - s["grad_entropy"][:, None] * p * (finite + entropy[:, None])
        grad[rows, at] += a[:, 0]
        return [logprob, entropy, grad]
    if case["top"] == 0:
        return [logprob, entropy]
    values, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    return [logprob, entropy, (values - torch.logsumexp(logits, 1, keepdim=True))[:, :case["top"]], ids[:, :case["top"]]]
