"""Gradients of the row-wise layers' activations where numbers leave their type's range (``cumm_amd.torch_layers``)."""
import math

import pytest
import torch

import layers_ref as R

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "sigmoid", "leaky_relu", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def L():
    from cumm_amd import torch_bridge, torch_layers
    assert torch_bridge._native() is not None
    return torch_layers


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n", [64, 136])      # few channels, and more, whose argument is kept in f16
@pytest.mark.parametrize("residual", [False, True])
def test_slopes_of_arguments_beyond_the_type(L, act, n, residual):
    """Arguments of +-90000, finite in 32 bits and infinite in f16: the slopes there are 0, 1 or the leak, whether the gradient that
    comes is zero or not, and the channels beside are as ever."""
    m, k, leak = 40, 8, 0.25
    x, w = torch.zeros(m, k, device="cuda", dtype=torch.float16), torch.zeros(n, k, device="cuda", dtype=torch.float16)
    x[:, 0], x[:, 1] = 60000, 1
    sign = torch.where(torch.arange(n, device="cuda") % 2 == 0, 1.0, -1.0)
    w[:, 0], w[n // 2:, 0], w[:, 1] = 1.5 * sign, 0, 0.5 * sign      # half of the channels are ordinary: +-0.5
    dy = torch.zeros(m, n, device="cuda", dtype=torch.float16)
    dy[:5] = 2.0 ** -8
    r = torch.zeros(m, n, device="cuda", dtype=torch.float16) if residual else None
    b = torch.zeros(n, device="cuda", dtype=torch.float16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(L.linear(*leaves, activation=act, residual=r, slope=leak), leaves, dy)
    with torch.no_grad():
        z = R.mm(x.double(), w.double())
        far = z.abs() > 1e4
        slope = R.slope(torch.where(far, z.sign() * 700, z), act, leak)      # (as at infinity)
        dz = dy.double() * slope
        # a slope is off by 2^-20, its product with the gradient rounded once, sums in 32 bits, rounded once; halves of the smallest step
        ddz = dy.double() * 2.0 ** -20 + dz.abs() * 2.0 ** -11 + 2.0 ** -25
        ax, aw = x.double(), w.double().abs()
        want = R.mm(dz, w.double().t()), R.mm(dz.t(), x.double().t()), dz.sum(0)
        errs = R.mm(ddz, aw.t()), R.mm(ddz.t(), ax.t()), ddz.sum(0)
        for name, a, e, err in zip(("grad_x", "grad_weight", "grad_bias"), got, want, errs):
            assert ((a.double() - e).abs() <= err * 1.01 + e.abs() * (2.0 ** -11 + 2.0 ** -16) + 2.0 ** -25).all(), name


@pytest.mark.parametrize("act", ["relu", "leaky_relu"])
@pytest.mark.parametrize("n", [64, 136])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("python", [False, True])
def test_infinite_gradients_stop_at_a_gate(L, monkeypatch, act, n, residual, python):
    """A gradient that is infinite (an overflow of scaled losses) is zero behind a closed ReLU, the leak times it behind a leaky one; one
    of an argument that is NaN passes."""
    if python:
        from cumm_amd import torch_bridge
        monkeypatch.setattr(torch_bridge, "_native_module", False)
    m, k, leak = 12, 8, 0.25
    x, w = (torch.zeros(r, k, device="cuda", dtype=torch.float16) for r in (m, n))
    x[:, 0] = torch.where(torch.arange(m, device="cuda") % 2 == 0, 1.0, -1.0)
    x[9, 0] = math.nan
    w[:, 0], w[:, 1] = 1, 2.0 ** -9
    b = torch.zeros(n, device="cuda", dtype=torch.float16)
    dy = torch.ones(m, n, device="cuda", dtype=torch.float16)
    dy[3, 5] = dy[4, 6] = math.inf      # behind a closed gate, and an open one
    r = torch.zeros(m, n, device="cuda", dtype=torch.float16) if residual else None
    leaves = [t.requires_grad_() for t in (x, w, b)]
    gx, _, gb = torch.autograd.grad(L.linear(*leaves, activation=act, residual=r, slope=leak), leaves, dy)
    off = 0.0 if act == "relu" else leak
    rows = [i for i in range(m) if i not in (3, 4)]
    passes = torch.where(torch.arange(m, device="cuda") % 2 == 0, 1.0, off)
    passes[9] = 1
    assert torch.equal(gx[rows, 1], (passes[rows] * n * 2.0 ** -9).half())
    assert float(gx[4, 1]) == math.inf and float(gx[3, 1]) == (0 if act == "relu" else math.inf)
    assert float(gb[6]) == math.inf and (act == "leaky_relu" or bool(gb[5].isfinite()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [64, 136])
def test_the_lower_tail_of_a_gelu(L, dtype, n):
    """Relative to the value, down to where bf16 ends: the result, and the slope by the gradient of x."""
    eps, tiny = {torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -134)}[dtype]
    z = -torch.linspace(0.5, 12.5, 3000, device="cuda").to(dtype).unique().flip(0)
    x, w = torch.zeros(z.numel(), 8, device="cuda", dtype=dtype), torch.zeros(n, 8, device="cuda", dtype=dtype)
    x[:, 0], w[0, 0] = z, 1      # (one channel is the argument, the others' is zero)
    dy = torch.zeros(z.numel(), n, device="cuda", dtype=dtype)
    dy[:, 0] = 1
    leaves = [t.requires_grad_() for t in (x, w)]
    out = L.linear(*leaves, activation="gelu")
    gx, = torch.autograd.grad(out, [x], dy)
    d = z.double()
    # the tail's quotient 1.6e-4 and its evaluation 2^-18; the exponent, of up to 113, is off by two roundings of 2^-24, times ln 2
    off = 1.7e-4 + 2.0 ** -18 + 113 * 2.0 ** -23 * 0.7
    want = d * 0.5 * torch.special.erfc(-d / math.sqrt(2))
    assert ((out[:, 0].double() - want).abs() <= want.abs() * (eps + off) * 1.01 + tiny).all()
    # the slope is tail + z density, of opposite signs: errors of both count; dz and grad_x are rounded
    density = torch.exp(-d * d / 2) / math.sqrt(2 * math.pi)
    slope = want / d + d * density
    allowed = (want / d * off + d.abs() * density * off) * 1.01
    assert ((gx[:, 0].double() - slope).abs() <= allowed + (slope.abs() * eps + tiny) * 2.02).all()
