"""Gradients over many rows, of whole numbers, bit for bit."""
import pytest
import torch

import whole_layers as W

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def L():
    from cumm_amd import torch_bridge, torch_layers
    assert torch_bridge._native() is not None
    return torch_layers


@pytest.mark.parametrize("m,k,n", W.NARROW + W.LARGE)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("act", ["none", "relu"])
def test_linear_loses_no_row(L, act, dtype, m, k, n):
    data = W.linear(m, k, n, "cuda")
    z, out, dz = W.linear_want(*data, act == "relu")
    x, w, b, r, dy = (t.to(dtype) for t in data)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    got = L.linear(x, w, b, activation=act, residual=r)
    grads = torch.autograd.grad(got, leaves, dy)
    want = [torch.mm(dz, data[1].float()), torch.mm(dz.t().contiguous(), data[0].float()), dz.sum(0), dy.float()]
    assert all(float(t.abs().max()) < 1 << 24 for t in want)
    for name, a, e in zip(("the result", "grad_x", "grad_weight", "grad_bias", "grad_residual"), (got,) + grads, [out] + want):
        assert torch.equal(a, e.to(dtype)), "%s: %d of %d" % (name, int((a != e.to(dtype)).sum()), a.numel())


@pytest.mark.parametrize("m,k", W.NORMS)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_loses_no_row(L, residual, dtype, m, k):
    """Of +-2 without an epsilon that counts, 1 / rms is 1/2 and u is x / 2; with k a power of two the mean is exact as well."""
    x, dy, ds = (t.to(dtype) for t in W.norm(m, k, "cuda"))
    w = torch.ones(k, device="cuda", dtype=dtype)
    u = x.float() / 2
    leaves = [(x / 2 if residual else x).requires_grad_(), w.requires_grad_()]
    if residual:      # 1 + 1
        r = (x / 2).detach().requires_grad_()
        out, total = L.rms_norm(leaves[0], w, 1e-12, residual=r)
        gx, gw, gr = torch.autograd.grad((out, total), leaves + [r], (dy, ds))
        assert torch.equal(total, x) and torch.equal(gx, gr)
    else:
        out = L.rms_norm(leaves[0], w, 1e-12)
        gx, gw = torch.autograd.grad(out, leaves, dy)
    assert torch.equal(out, u.to(dtype))
    assert torch.equal(gw, (dy.float() * u).sum(0).to(dtype))
    if k & (k - 1) == 0:
        want = (dy.float() - u * (dy.float() * u).mean(1, keepdim=True)) / 2
        if residual:
            want = want + ds.float()
        assert torch.equal(gx, want.to(dtype))


@pytest.mark.parametrize("m", [1, 7, 16])
@pytest.mark.parametrize("k,n", [(64, 4096), (64, 4104), (1000, 5001), (520, 8184), (4096, 8200)])
@pytest.mark.parametrize("dtype", HALVES + [torch.int8])
def test_few_rows_of_many_columns(L, dtype, m, k, n):
    """Both kernels for few rows, on either side of the line between them."""
    x, w, b, r, _ = W.linear(m, k, n, "cuda")
    want = torch.mm(x.float(), w.float().t().contiguous()) + b.float() + r.float()
    if dtype == torch.int8:
        one = lambda c: torch.ones(c, device="cuda")
        got = L.linear_s8(x, one(m), w, one(n), b.float(), residual=r.half(), dtype=torch.float16)
    else:
        got = L.linear(x.to(dtype), w.to(dtype), b.to(dtype), residual=r.to(dtype))
    assert torch.equal(got, want.to(got.dtype))
