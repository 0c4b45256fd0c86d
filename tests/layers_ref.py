"""The formulas of the row-wise layers in 64 bits."""
import math

import torch


def mm(a, b):
    """a [m, k] times the rows of b [n, k]"""
    return torch.mm(a.contiguous(), b.t().contiguous())


def act(z, name, slope):
    if name == "relu":
        return z.clamp_min(0)
    if name == "leaky_relu":
        return torch.where(z >= 0, z, z * slope)
    if name == "sigmoid":
        return torch.special.expit(z)
    if name == "silu":
        return z * torch.special.expit(z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return z * torch.special.expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def slope(z, name, leak):
    z = z.detach().clone().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(act(z, name, leak).sum(), z)[0]


def linear(x, w, bias, name, residual, leak):
    """(the activation's argument, the result)"""
    z = mm(x.detach().double(), w.detach().double())
    if bias is not None:
        z = z + bias.detach().double()
    out = act(z, name, leak)
    return z, out if residual is None else out + residual.detach().double()
