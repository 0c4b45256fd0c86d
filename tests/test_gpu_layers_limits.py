"""Row-wise layers of sizes near the limits of a launch."""
import pytest
import torch

import layers_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    from cumm_amd import torch_bridge, torch_layers
    assert torch_bridge._native() is not None
    return torch_layers


def whole(g, *shape):
    return torch.randint(-3, 4, shape, generator=g, device="cuda", dtype=torch.int8).half()


@pytest.mark.parametrize("m", [1, 17])
def test_linear_of_very_many_columns(L, m):
    """2^27 of them: whole numbers, so that every sum is exact."""
    n, k = 1 << 27, 8
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = whole(g, m, k), whole(g, n, k)
    if m > 1:
        n = (1 << 26) + 40
        w = w[:n]
    got = L.linear(x, w)
    for row in range(0, m, 8):
        want = torch.zeros(n, device="cuda")
        for j in range(k):
            want += x[row, j].float() * w[:, j].float()
        assert torch.equal(got[row], want.half())


def test_linear_of_very_many_rows(L):
    m, n, k = (1 << 30) + 77, 8, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = torch.zeros(m, k, device="cuda", dtype=torch.float16), whole(g, n, k)
    at = torch.cat([torch.arange(0, 300), torch.arange((1 << 29) - 100, (1 << 29) + 100), torch.arange(m - 300, m)]).cuda()
    x[at] = whole(g, at.numel(), k)
    got = L.linear(x, w)
    assert torch.equal(got[at].double(), R.mm(x[at].double(), w.double()))
    assert not bool(got[300:(1 << 29) - 100].any()) and not bool(got[(1 << 29) + 100:m - 300].any())


@pytest.mark.parametrize("k", [(1 << 28) + 24, (1 << 24) + 17])
def test_norm_of_one_very_long_row(L, k):
    """Elements of +-1 and +-2 in a row: the statistics are those of their counts."""
    g = torch.Generator(device="cuda").manual_seed(k)
    signs = lambda: (torch.randint(0, 2, (1, k), generator=g, device="cuda", dtype=torch.int8) * 2 - 1).half()
    x, w, dy = signs() * 2, torch.ones(k, device="cuda", dtype=torch.float16), signs()
    leaves = [t.requires_grad_() for t in (x, w)]
    out = L.rms_norm(*leaves, 1e-6)
    gx, gw = torch.autograd.grad(out, leaves, dy)
    with torch.no_grad():
        assert torch.equal(out, x / 2) and torch.equal(gw, (x / 2 * dy)[0])
        # u = x / 2, grad_x = (dy - u mean(dy u)) / 2: the mean, of a sum in 32 bits of k terms, is off by no more than k 2^-24; one rounding
        mean = float((dy * (x / 2)).double().mean())
        want = (dy.float() - x / 2 * mean) / 2
        # sums of a thread's share, then of the threads': k / 1024 + 1024 additions
        allowed = (k / 1024 + 1024) * 2.0 ** -24 / 2 + 2.0 ** -12
        assert float((gx.float() - want).abs().max()) <= allowed


@pytest.mark.parametrize("python", [False, True])
def test_rows_very_far_apart(L, monkeypatch, python):
    """Columns of a matrix whose rows are 8 MiB and more: copied, for the gradient of the result too."""
    if python:
        from cumm_amd import torch_bridge
        monkeypatch.setattr(torch_bridge, "_native_module", False)
    g = torch.Generator(device="cuda").manual_seed(2)
    for columns in ((4 << 20) - 1, 4 << 20, 5 << 20):
        wide = torch.zeros(6, columns, device="cuda", dtype=torch.float16)
        wide[:, 8:280] = whole(g, 6, 272)
        for n in (64, 136):
            w, norm = whole(g, n, 136), whole(g, 136)
            x, dy, r = wide[:, 8:144], wide[:, 144:144 + n], wide[:, 140:140 + n]
            near = [t.contiguous() for t in (x, dy, r)]
            for act in ("none", "relu"):
                step = lambda x, dy, r: (L.linear(x, w, activation=act, residual=r),) + torch.autograd.grad(
                    L.linear(x.requires_grad_(), w.requires_grad_(), activation=act, residual=r), (x, w), dy)
                assert all(torch.equal(a, b) for a, b in zip(step(x.detach(), dy, r), step(near[0].detach(), *near[1:])))
            assert torch.equal(L.rms_norm(x, norm), L.rms_norm(near[0], norm))
            assert all(torch.equal(a, b) for a, b in zip(L.quantize_rows(x), L.quantize_rows(near[0])))
