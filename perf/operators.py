"""Cases of the row-wise layers: a matrix product with bias, activation and residual in its epilogue (two-byte and 8-bit
operands, one token to thousands, with its gradients), the root-mean-square norm with the residual's addition (its output
in the type of its input or in 8 bits with a scale per row, with its gradients) and the quantisation of rows to 8 bits.

``run`` computes a case in plain torch operations, or, where ``own`` is true, by the calls that a program makes of
``cumm_amd.torch_layers``.  ``exact`` is the definition in 64 bits.

8-bit results are the whole numbers themselves, beside the scale of their row: code * scale is the value.  A code is the
whole number next to 127 v / max |v| of its row, ties to even, v exact in 32 bits: it depends on no order of a sum.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # the widening product of a feed-forward block, a batch of 8192 rows
        dict(name="linear large", op="linear", type="bf16", m=8192, k=4096, n=4096, act="gelu_tanh", bias=True, residual=True),
        # no size a multiple of anything: the rows of neither operand begin at whole words
        dict(name="linear odd", op="linear", type="f16", m=2001, k=1163, n=777, act="relu", bias=True, residual=False),
        # one token: the weight is read once, nothing else counts
        dict(name="linear one token", op="linear", type="bf16", m=1, k=4096, n=16384, act="silu", bias=False, residual=False),
        # a training step of the widening product: result and every gradient
        dict(name="linear train", op="linear_train", type="bf16", m=4096, k=2048, n=8192, act="gelu", bias=True, residual=False),
        # a training step of a point-wise layer on the voxels of one frame: few channels, very many rows
        dict(name="linear train voxels", op="linear_train", type="f16", m=119985, k=64, n=128, act="relu", bias=True, residual=True),
        # inference in 8 bits, a batch of 8192 rows
        dict(name="linear s8 large", op="linear_s8", type="bf16", m=8192, k=4096, n=8192, act="silu", bias=True, residual=False),
        # inference in 8 bits, sixteen sequences at a token each
        dict(name="linear s8 few tokens", op="linear_s8", type="f16", m=16, k=8192, n=4096, act="none", bias=True, residual=True),
        # the norm in front of a block, the residual stream carried along
        dict(name="norm large", op="norm", type="bf16", m=16384, k=4096, residual=True),
        # the same with its output in 8 bits, an odd number of rows
        dict(name="norm s8", op="norm_s8", type="bf16", m=8191, k=5120, residual=True),
        # a training step of the norm
        dict(name="norm train", op="norm_train", type="f16", m=8192, k=2048, residual=True),
        # activations to 8 bits between two products
        dict(name="quantize large", op="quantize", type="bf16", m=8192, k=8192),
        # the same for one token: a call's latency
        dict(name="quantize one token", op="quantize", type="f16", m=1, k=11000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _channels(rng, lo, hi):
    """A number of channels: a multiple of 64, of 8, or any."""
    c, step = _log(rng, lo, hi), rng.choice([64, 64, 8, 1])
    return max(step, c // step * step)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_train", "linear_s8", "norm", "norm_s8", "norm_train", "quantize"])
    most = max(work(c)["flops"] for c in listed() if c["op"] == op)
    bytes_most = max(work(c)["bytes"] for c in listed() if c["op"] == op)
    while True:
        case = dict(op=op, type=rng.choice(["f16", "bf16"]))
        if op.startswith("linear"):
            case |= dict(m=_log(rng, 16, 120000) if op == "linear_train" else _log(rng, 1, 16384), k=_channels(rng, 32, 8192),
                         n=_channels(rng, 32, 16384), act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                         bias=rng.random() < 0.7, residual=rng.random() < 0.5)
        elif op == "quantize":
            case |= dict(type=rng.choice(["f16", "bf16", "f32"]), m=_log(rng, 1, 30000), k=_channels(rng, 32, 20000))
        else:
            case |= dict(m=_log(rng, 1, 30000), k=_channels(rng, 32, 16384), residual=rng.random() < 0.7)
        w = work(case)
        if w["flops"] <= most and w["bytes"] <= bytes_most:
            return case


def _rng(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(dtype)


def _activations(g, m, k, dtype):
    """Rows as a residual stream has them: of unlike size, with some channels that stand out."""
    x = torch.randn((m, k), generator=g, device=DEVICE)
    x *= torch.exp(0.5 * torch.randn((m, 1), generator=g, device=DEVICE))
    x *= 1 + 8 * (torch.rand((1, k), generator=g, device=DEVICE) < 0.01)
    return x.to(dtype)


def prepare(case, seed):
    g, op, dtype, m, k = _rng(seed), case["op"], TYPES[case["type"]], case["m"], case["k"]
    s = dict(case=case)
    if op.startswith("linear"):
        n = case["n"]
        if op == "linear_s8":      # what the norm in 8 bits has left, and a weight that is kept in 8 bits
            s["x"] = (32 * torch.randn((m, k), generator=g, device=DEVICE)).round().clamp(-127, 127).to(torch.int8)
            s["weight"] = (40 * torch.randn((n, k), generator=g, device=DEVICE)).round().clamp(-127, 127).to(torch.int8)
            s["x_scale"] = (0.5 + torch.rand(m, generator=g, device=DEVICE)) / 32
            s["weight_scale"] = (0.5 + torch.rand(n, generator=g, device=DEVICE)) / (40 * math.sqrt(k))
            s["bias"] = _normal(g, (n,), torch.float32, 0.2) if case["bias"] else None
        else:
            s["x"] = _normal(g, (m, k), dtype)
            s["weight"] = _normal(g, (n, k), dtype, 1 / math.sqrt(k))
            s["bias"] = _normal(g, (n,), dtype, 0.2) if case["bias"] else None
        s["residual"] = _normal(g, (m, n), dtype) if case["residual"] else None
        if op == "linear_train":
            s["grad"] = _normal(g, (m, n), dtype)
    else:
        s["x"] = _activations(g, m, k, dtype)
        if op != "quantize":
            s["weight"] = _normal(g, (k,), torch.float32, 0.2).add_(1).to(dtype)
            s["residual"] = _activations(g, m, k, dtype) if case["residual"] else None
        if op == "norm_train":
            s["grad"] = _normal(g, (m, k), dtype)
            s["grad_sum"] = _normal(g, (m, k), dtype) if case["residual"] else None
    if op.endswith("train"):      # leaves, as a program's parameters are
        for name in ("x", "weight", "bias", "residual"):
            if s.get(name) is not None:
                s[name].requires_grad_()
    return s


# ---- the plain forms

def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _codes(v):
    """(whole numbers, 32-bit largest magnitude) of the rows of v: the quotient in 64 bits, where ties are ties."""
    top = v.abs().amax(1, keepdim=True)
    t = v.double() * 127 / torch.where(top > 0, top, torch.ones_like(top)).double()
    return torch.round(t).to(torch.int8), top[:, 0]


def _plain(s):
    case = s["case"]
    op, dtype = case["op"], TYPES[case["type"]]
    s = {k: v.detach() if torch.is_tensor(v) else v for k, v in s.items()}
    x = s["x"].float()
    if op.startswith("linear"):
        z = x @ s["weight"].float().t()
        if op == "linear_s8":
            z = z * s["x_scale"][:, None] * s["weight_scale"]
        if s["bias"] is not None:
            z = z + s["bias"].float()
        out = _act(z, case["act"])
        if s["residual"] is not None:
            out = out + s["residual"].float()
        out = out.to(dtype)
        if op != "linear_train":
            return out
        dz = s["grad"].float() * _act_slope(z, case["act"])
        return dict(out=out, grad_x=(dz @ s["weight"].float()).to(dtype), grad_weight=(dz.t() @ x).to(dtype),
                    grad_bias=dz.sum(0).to(dtype) if s["bias"] is not None else None,
                    grad_residual=s["grad"] if s["residual"] is not None else None)
    if op == "quantize":
        codes, top = _codes(x)
        return dict(codes=codes, scale=top / 127)
    h = x
    if s["residual"] is not None:
        total = (x + s["residual"].float()).to(dtype)
        h = total.float()
    inv = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    res = dict(total=total) if s["residual"] is not None else {}
    w = s["weight"].float()
    if op == "norm_s8":
        codes, top = _codes(h * w)
        return dict(res, codes=codes, scale=top * inv[:, 0] / 127)
    res["out"] = (h * inv * w).to(dtype)
    if op == "norm_train":
        u, g = h * inv, s["grad"].float()
        gw = g * w
        dh = inv * (gw - u * (gw * u).mean(1, keepdim=True))
        if s["grad_sum"] is not None:
            dh = dh + s["grad_sum"].float()
        dh = dh.to(dtype)
        res |= dict(grad_x=dh, grad_weight=(g * u).sum(0).to(dtype))
        if s["residual"] is not None:
            res["grad_residual"] = dh
    return res


# ---- the framework's calls

def _own(s):
    from cumm_amd import torch_layers as L
    case = s["case"]
    op = case["op"]
    if op == "linear":
        return L.linear(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"])
    if op == "linear_s8":
        return L.linear_s8(s["x"], s["x_scale"], s["weight"], s["weight_scale"], s["bias"], activation=case["act"],
                           residual=s["residual"], dtype=TYPES[case["type"]])
    if op == "linear_train":
        names = [name for name in ("x", "weight", "bias", "residual") if s[name] is not None]
        out = L.linear(s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"])
        grads = torch.autograd.grad(out, [s[name] for name in names], s["grad"])
        return dict({"grad_" + name: g for name, g in zip(names, grads)}, out=out.detach())
    if op == "quantize":
        codes, scale = L.quantize_rows(s["x"])
        return dict(codes=codes, scale=scale)
    if op == "norm_s8":
        got = L.rms_norm_s8(s["x"], s["weight"], EPS, residual=s["residual"])
        return dict(zip(("codes", "scale", "total"), got))
    got = L.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"])
    if s["residual"] is None:
        got = (got,)
    res = dict(zip(("out", "total"), got))
    if op == "norm_train":
        names = [name for name in ("x", "weight", "residual") if s[name] is not None]
        grads = torch.autograd.grad(got, [s[name] for name in names], [s["grad"], s["grad_sum"]][:len(got)])
        res = {name: t.detach() for name, t in res.items()}
        res |= {"grad_" + name: g for name, g in zip(names, grads)}
    return res


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without

def work(case):
    op, m, k = case["op"], case["m"], case["k"]
    size = 4 if case["type"] == "f32" else 2
    if op.startswith("linear"):
        n = case["n"]
        operands = (m * k + n * k) * (1 if op == "linear_s8" else 2)
        more = 2 * n * case["bias"] + 2 * m * n * case["residual"] + (4 * (m + n) if op == "linear_s8" else 0)
        if op != "linear_train":
            return dict(bytes=operands + more + 2 * m * n, flops=2.0 * m * n * k)
        # result and gradients written once, the gradient of the result read once (it is the residual's, as it is)
        return dict(bytes=2 * operands + more + 2 * n * case["bias"] + 2 * 2 * m * n, flops=6.0 * m * n * k)
    carried = 2 if op != "quantize" and case["residual"] else 0      # the residual read, the sum written
    if op == "quantize":
        return dict(bytes=m * k * (size + 1) + 4 * m, flops=4.0 * m * k)
    if op == "norm_s8":
        return dict(bytes=m * k * (size * (1 + carried) + 1) + 4 * m + size * k, flops=8.0 * m * k)
    if op == "norm":
        return dict(bytes=m * k * size * (2 + carried) + size * k, flops=5.0 * m * k)
    # both directions: two gradients in, one out (it is the residual's too)
    return dict(bytes=m * k * size * (2 + carried + 2 + carried // 2) + 2 * size * k, flops=16.0 * m * k)


# ---- the definitions in 64 bits

def _exact_act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z * torch.special.expit(z)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    return z * torch.special.expit(2 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))


def exact(case, seed):
    s = prepare(case, seed)
    op, dtype = case["op"], TYPES[case["type"]]
    d = {name: t.detach().to(torch.float64) for name, t in s.items() if torch.is_tensor(t)}
    leaves = [name for name in ("x", "weight", "bias", "residual") if name in d]
    if op.endswith("train"):
        for name in leaves:
            d[name].requires_grad_()
    with torch.set_grad_enabled(op.endswith("train")):
        if op.startswith("linear"):
            x = d["x"] * d["x_scale"].unsqueeze(1) if op == "linear_s8" else d["x"]
            w = d["weight"] * d["weight_scale"].unsqueeze(1) if op == "linear_s8" else d["weight"]
            z = torch.mm(x, w.transpose(0, 1).contiguous())
            out = _exact_act(z + d["bias"] if "bias" in d else z, case["act"])
            out = out + d["residual"] if "residual" in d else out
            if op != "linear_train":
                return out
            grads = torch.autograd.grad(out, [d[name] for name in leaves], d["grad"])
            return dict({"grad_" + name: g for name, g in zip(leaves, grads)}, out=out.detach())
        if op == "quantize":
            return dict(codes=None, scale=d["x"].abs().max(dim=1).values / 127)
        res = {}
        h = d["x"]
        if "residual" in d:
            total = d["x"] + d["residual"]
            res["total"] = total.detach()
            # the norm is that of the sum as it is stored
            h = total + (s["x"].detach().float() + s["residual"].detach().float()).to(dtype).double() - total.detach()
        u = h / torch.sqrt(h.pow(2).sum(1, keepdim=True) / case["k"] + EPS)
        out = u * d["weight"]
        if op == "norm_s8":
            return dict(res, codes=None, scale=out.abs().max(dim=1).values / 127)
        res["out"] = out.detach()
        if op == "norm_train":
            through, came = ([out, total], [d["grad"], d["grad_sum"]]) if "residual" in d else ([out], [d["grad"]])
            grads = torch.autograd.grad(through, [d[name] for name in leaves], came)
            res |= {"grad_" + name: g for name, g in zip(leaves, grads)}
        return res
