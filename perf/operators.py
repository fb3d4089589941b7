"""The 8-bit row operators at the sizes they are used at: cases, their plain forms, and their definition in 64 bits.

Rows held in 8 bits: row r of a matrix is q[r, :] * scale[r], q int8 in [-127, 127] (round to nearest even), scale[r] = max|row| / 127.

    norm      h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight; y in 8-bit rows, and for training h in 8-bit rows too
    linear    z = A B^T for A and B in 8-bit rows (tokens and output channels) + bias
    backward  the linear's gradients: grad B^T = grad_A, grad^T A = grad_B, A being the activations kept in 8 bits
    normback  the norm's gradients from h kept in 8 bits
    block     norm and linear as a decoder calls them, from x to z
    step      norm, linear and both gradients through autograd, as a training step calls them

`own` False: elementary torch operations in 32 bits.  `own` True: the calls a user makes of the framework.
"""
import os
import sys

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a decoder: latency
        {"name": "norm one token", "op": "norm", "rows": 1, "cols": 4096, "type": "bf16", "save": False},
        # a ragged batch of prompts in f32, every step's activations kept
        {"name": "norm ragged f32", "op": "norm", "rows": 1777, "cols": 1111, "type": "f32", "save": True},
        # a training batch, with the checkpoint
        {"name": "norm training batch", "op": "norm", "rows": 8192, "cols": 8192, "type": "bf16", "save": True},
        # one token through a projection: the weights' read
        {"name": "linear one token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": False},
        # a short prompt of odd length, odd widths, with a bias
        {"name": "linear odd", "op": "linear", "m": 333, "n": 1531, "k": 1111, "type": "f32", "bias": True},
        # a long prompt through a wide projection
        {"name": "linear prompt", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "bias": False},
        # a small f32 layer's gradients (512 x 256, the batched matrices of this framework's training workload)
        {"name": "backward small f32", "op": "backward", "m": 512, "n": 512, "k": 256, "type": "f32"},
        # a wide layer's gradients
        {"name": "backward training batch", "op": "backward", "m": 8192, "n": 8192, "k": 4096, "type": "bf16"},
        # the norm's gradients: a few odd rows, and a training batch
        {"name": "normback odd f16", "op": "normback", "rows": 77, "cols": 1001, "type": "f16"},
        {"name": "normback training batch", "op": "normback", "rows": 8192, "cols": 8192, "type": "bf16"},
        # sixteen sequences decoding together
        {"name": "block sixteen tokens", "op": "block", "m": 16, "n": 8192, "k": 4096, "type": "bf16"},
        # a whole training step of a layer
        {"name": "step", "op": "step", "m": 4096, "n": 4096, "k": 4096, "type": "bf16"},
    ]


def draw(rng):
    def size(lo, hi):
        v = int(round(lo * (hi / lo) ** rng.random()))
        if rng.random() < 0.5 and v >= 64:
            v = v // 32 * 32
        return v if v != 3072 else v + 1

    op = rng.choice(["norm", "linear", "linear", "backward", "normback", "block", "step"])
    if op in ("norm", "normback"):
        case = {"op": op, "rows": size(1, 8192), "cols": size(64, 8192), "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
        if op == "norm":
            case["save"] = rng.random() < 0.5
    elif op == "linear":
        case = {"op": op, "m": size(1, 8192), "n": size(64, 8192), "k": size(64, 8192), "type": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "bias": rng.random() < 0.3}
    elif op == "backward":
        case = {"op": op, "m": size(1, 8192), "n": size(64, 8192), "k": size(64, 4096), "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
    elif op == "block":
        case = {"op": op, "m": size(1, 256), "n": size(64, 8192), "k": size(64, 8192), "type": rng.choice(["bf16", "f16"])}
    else:
        case = {"op": op, "m": size(16, 4096), "n": size(64, 4096), "k": size(64, 4096), "type": rng.choice(["bf16", "bf16", "f16"])}
    return case


def work(case):
    e = BYTES[case["type"]]
    if case["op"] in ("norm", "normback"):
        n = case["rows"] * case["cols"]
        if case["op"] == "norm":  # x, residual, h, q and the values it stands for; with the checkpoint, its q and values
            return {"bytes": n * (3 * e + 3 + (3 if case["save"] else 0)) + case["cols"] * e + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": n * (3 * e + 1) + 2 * case["cols"] * e + 8 * case["rows"], "flops": 10 * n}  # grad, grad_h, checkpoint; grad_x
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "linear":
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * e, "flops": 2 * m * n * k}
    if case["op"] == "backward":
        return {"bytes": m * n * e + (m * k + n * k) * (1 + e) + 4 * (m + n), "flops": 4 * m * n * k}
    if case["op"] == "block":
        return {"bytes": 3 * m * k * e + n * k + 4 * n + m * n * e, "flops": 2 * m * n * k}
    # x, residual, h, weight, z; grad of z and of h, the gradients of x and of the weight
    return {"bytes": e * (5 * m * k + 2 * n * k + 2 * m * n), "flops": 6 * m * n * k}


# --------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def hidden(rows, cols):  # hidden states: a few channels are much larger than the others
        wide = torch.where(torch.rand(cols, generator=g, device="cuda") < 0.01, 8.0, 1.0)
        return normal(rows, cols) * wide

    def rows8(rows, cols, size):  # what a quantisation leaves: the largest value of a row is 127
        v = normal(rows, cols)
        top = v.abs().amax(1, keepdim=True)
        q = torch.round(v * (127 / top)).to(torch.int8)
        return q, (top[:, 0] * (size / 127) * (0.5 + torch.rand(rows, generator=g, device="cuda")))

    s = {"case": dict(case)}
    if case["op"] == "norm":
        s["x"], s["residual"] = normal(case["rows"], case["cols"]).to(t), hidden(case["rows"], case["cols"]).to(t)
        s["x"][3::97] = 0  # padding tokens
        s["residual"][3::97] = 0
        s["weight"] = (1 + 0.2 * normal(case["cols"])).to(t)
    elif case["op"] == "normback":
        r, c = case["rows"], case["cols"]
        s["weight"] = (1 + 0.2 * normal(c)).to(t)
        s["q"], s["scale"] = rows8(r, c, 1.0)
        s["rstd"] = torch.rsqrt((s["q"].float() * s["scale"][:, None]).square().mean(1) + EPS)
        s["grad"], s["grad_h"] = normal(r, c).to(t), normal(r, c).to(t)
    elif case["op"] in ("linear", "backward"):
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["a_scale"] = rows8(m, k, 1.0)
        s["b"], s["b_scale"] = rows8(n, k, k ** -0.5)
        if case["op"] == "linear":
            s["bias"] = normal(n).to(t) if case["bias"] else None
        else:
            s["grad"] = normal(m, n).to(t)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["x"], s["residual"] = normal(m, k).to(t), hidden(m, k).to(t)
        s["weight"] = (1 + 0.2 * normal(k)).to(t)
        if case["op"] == "block":
            s["b"], s["b_scale"] = rows8(n, k, k ** -0.5)
        else:
            s["w"] = (normal(n, k) * k ** -0.5).to(t)
            s["grad_z"], s["grad_h"] = normal(m, n).to(t), normal(m, k).to(t)
            for name in ("x", "residual", "weight", "w"):
                s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------ plain form
def _quantize(y):
    scale = y.abs().amax(1) / 127
    q = torch.round(y / torch.where(scale > 0, scale, 1.0)[:, None])
    return q, scale


def _values(q, scale):
    return q.float() * scale[:, None]


def _norm(x, residual, weight):
    h = x.float() + residual.float()
    rstd = torch.rsqrt(h.square().mean(1) + EPS)
    return h, rstd, h * rstd[:, None] * weight.float()


def _norm_back(grad, values, rstd, weight, grad_h):
    unit = values * rstd[:, None]
    inner = grad * weight.float()
    grad_x = rstd[:, None] * (inner - unit * (inner * unit).mean(1, keepdim=True)) + grad_h.float()
    return grad_x, (grad * unit).sum(0)


def _plain(s):
    case = s["case"]
    t = TYPES[case["type"]]
    if case["op"] == "norm":
        h, rstd, y = _norm(s["x"], s["residual"], s["weight"])
        out = [h.to(t), _values(*_quantize(y)).to(torch.bfloat16)]
        return out + [_values(*_quantize(h)).to(torch.bfloat16), rstd] if case["save"] else out
    if case["op"] == "normback":
        grad_x, grad_w = _norm_back(s["grad"].float(), _values(s["q"], s["scale"]), s["rstd"], s["weight"], s["grad_h"])
        return [grad_x.to(t), grad_w.to(t)]
    if case["op"] == "linear":
        z = (s["a"].float() @ s["b"].float().t()) * s["a_scale"][:, None] * s["b_scale"]
        return (z if s["bias"] is None else z + s["bias"].float()).to(t)
    if case["op"] == "backward":
        g = s["grad"].float()
        return [(g @ _values(s["b"], s["b_scale"])).to(t), (g.t() @ _values(s["a"], s["a_scale"])).to(t)]
    with torch.no_grad():
        h, rstd, y = _norm(s["x"], s["residual"], s["weight"])
        a, a_scale = _quantize(y)
        if case["op"] == "block":
            return [((a @ s["b"].float().t()) * a_scale[:, None] * s["b_scale"]).to(t), h.to(t)]
        b, b_scale = _quantize(s["w"].float())
        z = (a @ b.t()) * a_scale[:, None] * b_scale
        g = s["grad_z"].float()
        grad_y, grad_w = g @ _values(b, b_scale), g.t() @ _values(a, a_scale)
        grad_x, grad_norm = _norm_back(grad_y, _values(*_quantize(h)), rstd, s["weight"], s["grad_h"])
        return [z.to(t), h.to(t), grad_x.to(t), grad_norm.to(t), grad_w.to(t)]


# --------------------------------------------------------------------------------------------------- the framework's calls
def _package():
    if "tropical_gemm" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "tropical-gemm_b200"))
    import tropical_gemm.pytorch
    import tropical_gemm.rows8
    return tropical_gemm.rows8, tropical_gemm.pytorch


def _own(s):
    rows8, autograd = _package()
    case = s["case"]
    t = TYPES[case["type"]]
    if case["op"] == "norm":
        r = rows8.rmsnorm(s["x"], s["weight"], residual=s["residual"], eps=EPS, checkpoint=case["save"])
        out = [r.h, rows8.dequantize(r.rows, torch.bfloat16)]
        return out + [rows8.dequantize(r.checkpoint, torch.bfloat16), r.rstd] if case["save"] else out
    if case["op"] == "normback":
        return list(rows8.rmsnorm_backward(s["grad"], rows8.Rows8(s["q"], s["scale"]), s["rstd"], s["weight"], grad_h=s["grad_h"]))
    if case["op"] == "linear":
        return rows8.matmul(rows8.Rows8(s["a"], s["a_scale"]), rows8.Rows8(s["b"], s["b_scale"]), bias=s["bias"], dtype=t)
    if case["op"] == "backward":
        return list(rows8.matmul_backward(s["grad"], rows8.Rows8(s["a"], s["a_scale"]), rows8.Rows8(s["b"], s["b_scale"])))
    if case["op"] == "block":
        r = rows8.rmsnorm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return [rows8.matmul(r.rows, rows8.Rows8(s["b"], s["b_scale"]), dtype=t), r.h]
    z, h = autograd.rmsnorm_linear_rows8(s["x"], s["weight"], s["w"], residual=s["residual"], eps=EPS)
    grad_x, _, grad_norm, grad_w = torch.autograd.grad((z, h), (s["x"], s["residual"], s["weight"], s["w"]), (s["grad_z"], s["grad_h"]))
    return [z, h, grad_x, grad_norm, grad_w]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    s = {k: v.detach().double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}

    def held(v):  # the values that 8-bit rows of v stand for
        step = v.abs().max(dim=1, keepdim=True).values / 127
        return torch.where(step > 0, torch.round(v / step.clamp_min(1e-300)) * step, torch.zeros_like(v))

    def unit_of(h):
        return (h.pow(2).sum(dim=1, keepdim=True) / h.shape[1] + EPS).pow(-0.5)

    def norm_gradients(grad, h, rstd, weight, grad_h):
        u = h * rstd
        c = torch.einsum("ij,j,ij->i", grad, weight, u) / h.shape[1]
        return grad_h + (grad * weight - u * c[:, None]) * rstd, torch.einsum("ij,ij->j", grad, u)

    op = case["op"]
    if op == "norm":
        h = s["x"] + s["residual"]
        rstd = unit_of(h)
        out = [h, held(h * rstd * s["weight"])]
        return out + [held(h), rstd[:, 0]] if case["save"] else out
    if op == "normback":
        return list(norm_gradients(s["grad"], s["q"] * s["scale"][:, None], s["rstd"][:, None], s["weight"], s["grad_h"]))
    if op in ("linear", "backward"):
        a, b = torch.diag_embed(s["a_scale"]) @ s["a"] if case["m"] <= 64 else s["a"] * s["a_scale"][:, None], s["b"] * s["b_scale"][:, None]
        if op == "backward":
            return [torch.mm(s["grad"], b), torch.mm(s["grad"].T, a)]
        z = torch.mm(a, b.T)
        return z if s["bias"] is None else z + s["bias"][None]
    h = s["x"] + s["residual"]
    rstd = unit_of(h)
    a = held(h * rstd * s["weight"])
    if op == "block":
        return [torch.mm(a, (s["b"] * s["b_scale"][:, None]).T), h]
    b = held(s["w"])
    grad_x, grad_norm = norm_gradients(torch.mm(s["grad_z"], b), held(h), rstd, s["weight"], s["grad_h"])
    return [torch.mm(a, b.T), h, grad_x, grad_norm, torch.mm(s["grad_z"].T, a)]
