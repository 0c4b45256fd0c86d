"""Activations with a kink (``cumm_amd.torch_layers``): on which side of it an argument lies is a matter of its sign alone, so
layers of few channels decide it by the sum in 64 bits where the one in 32 lies within its own error of zero, the result and the
gradient alike.  All numbers here are exact in 32 bits once the gates are right, so results are compared bit for bit."""
import ctypes

import pytest
import torch

import layers_ref as R

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
TINY, STEP, LEAK = 2.0 ** -13, 2.0 ** -8, 0.25


@pytest.fixture(scope="module")
def L():
    from cumm_amd import torch_bridge, torch_layers
    assert torch_bridge._native() is not None
    return torch_layers


def cancelling(m, k, n, dtype, seed, pad=0, lead=0):
    """x and weight whose products are whole numbers up to 4080 that cancel, and one of +-2^-13: the argument is that one, and a sum of
    32 bits loses it against the others' partial sums wherever it does not come last."""
    g = torch.Generator().manual_seed(seed)
    h = (k - 1) // 2
    whole = torch.randint(128, 256, (m, h), generator=g) * 16 * (torch.randint(0, 2, (m, h), generator=g) * 2 - 1)
    signs = torch.randint(0, 2, (n, h), generator=g) * 2 - 1
    x, w = torch.zeros(m, k, dtype=torch.float64), torch.zeros(n, k, dtype=torch.float64)
    x[:, :h], x[:, h:2 * h] = whole.double(), -whole.double()
    w[:, :h], w[:, h:2 * h] = signs.double(), signs.double()
    x[:, 2 * h] = TINY * (torch.randint(0, 2, (m,), generator=g) * 2 - 1)
    w[:, 2 * h] = (torch.randint(0, 2, (n,), generator=g) * 2 - 1).double()
    order = torch.randperm(k, generator=g)

    def placed(t):
        field = torch.zeros(t.shape[0] * (k + pad) + lead, dtype=dtype, device="cuda")
        at = field[lead:].view(t.shape[0], k + pad)[:, :k]
        at.copy_(t[:, order].to(dtype))
        return at
    return placed(x), placed(w), x @ w.t()


@pytest.mark.parametrize("m,k,n", [(1, 24, 8), (17, 64, 128), (300, 120, 72), (2000, 128, 128), (700, 64, 64), (1000, 128, 40), (5, 8, 8)])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("act", ["relu", "leaky_relu"])
def test_gates_go_by_the_exact_argument(L, act, dtype, m, k, n):
    for pad, lead, residual in ((0, 0, False), (0, 0, True), (3, 5, False)):
        x, w, z = cancelling(m, k, n, dtype, m + k + n + lead, pad, lead)
        z = z.cuda()
        assert (z.abs() == TINY).all()
        b = torch.zeros(n, dtype=dtype, device="cuda")
        r = torch.zeros(m, n, dtype=dtype, device="cuda") if residual else None
        leaves = [t.requires_grad_() for t in (x.detach(), w.detach(), b)]
        out = L.linear(*leaves, activation=act, residual=r, slope=LEAK)
        off = 0.0 if act == "relu" else LEAK
        assert torch.equal(out.double(), torch.where(z > 0, z, z * off))
        dz = torch.where(z > 0, STEP, STEP * off).double()
        grads = torch.autograd.grad(out, leaves, torch.full_like(out, STEP))
        want = R.mm(dz, w.detach().double().t()), R.mm(dz.t(), x.detach().double().t()), dz.sum(0)
        for name, got, exact in zip(("grad_x", "grad_weight", "grad_bias"), grads, want):
            assert torch.equal(got, exact.to(dtype)), name


@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (129, 40, 24), (300, 128, 128)])
def test_what_the_activation_got_and_a_residual_in_the_result_s_place(L, m, k, n):
    """The interface below: pre_act, and out that is the residual; nothing beside the rows is written."""
    from cumm_amd import _capi
    for dtype, code in ((torch.float16, 7), (torch.bfloat16, 12)):
        x, w, z = cancelling(m, k, n, dtype, m)
        g = torch.Generator().manual_seed(m)
        res = torch.randint(-3, 4, (m, n), generator=g).double().cuda() * TINY
        out, pre = (torch.full((m, n + 16), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        out[:, 8:8 + n] = res.to(dtype)
        inner = out[:, 8:8 + n]
        a = _capi.LinearArgs(dtype=code, out_dtype=code, m=m, n=n, k=k, x=x.data_ptr(), weight=w.data_ptr(), out=inner.data_ptr(), residual=inner.data_ptr(),
                             pre_act=pre[:, 8:].data_ptr(), ld_x=k, ld_weight=k, ld_out=n + 16, ld_residual=n + 16, ld_pre_act=n + 16, act_type=1)
        assert _capi.lib().cumm_hip_linear_workspace(ctypes.byref(a)) == 0
        _capi.check(_capi.lib().cumm_hip_linear(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
        z = z.cuda()
        assert torch.equal(inner.double(), z.clamp_min(0) + res) and torch.equal(pre[:, 8:8 + n].double(), z)
        for t in (out, pre):
            assert (t[:, :8] == 7).all() and (t[:, 8 + n:] == 7).all()


def test_rows_of_zeros_and_numbers_without_a_bound(L):
    """No row of zeros is added up again for ever, an infinity or a NaN stays in its row, and lengths that overflow lose nothing."""
    for m, k, n in ((40, 64, 128), (300, 128, 64)):
        g = torch.Generator(device="cuda").manual_seed(k)
        x, w = (torch.randn(r, k, generator=g, device="cuda").bfloat16() for r in (m, n))
        x[7], x[9, 3], x[11, 5] = 0, float("nan"), float("inf")
        x[13] = x[13] * 2.0 ** 100      # (its square is beyond 32 bits)
        b = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        out = L.linear(*leaves, activation="relu")
        gx, = torch.autograd.grad(out, [x], torch.ones_like(out))
        with torch.no_grad():
            z = R.mm(x.double(), w.double())
            assert (out[7] == 0).all() and (gx[7] == 0).all()
            assert out[9].isnan().all()
            passes = ~(z <= 0)      # (a NaN does)
            assert torch.equal(out != 0, passes)
            want, mag = R.mm(passes.double(), w.double().t()), R.mm(passes.double(), w.double().abs().t())
            # a sum of n products in 32 bits, rounded once
            assert ((gx.double() - want).abs() <= (n + 8) * 2.0 ** -23 * mag * 1.01 + want.abs() * 2.0 ** -8 + 2.0 ** -134).all()


@pytest.mark.parametrize("m,k,n", [(1, 8, 8), (129, 64, 72), (300, 128, 40)])
@pytest.mark.parametrize("act", [1, 3])
def test_the_backward_pass_without_a_gate(L, act, m, k, n):
    """Below torch: nobody has kept the forward pass's gate, a launch before makes it; it and the workspace end where they should."""
    from cumm_amd import _capi
    lib = _capi.lib()
    x, w, _ = cancelling(m, k, n, torch.float16, m)
    dy = torch.full((m, n), STEP, device="cuda", dtype=torch.float16)
    stream = torch.cuda.current_stream().cuda_stream
    size = m * _capi.LINEAR_GATE_BYTES(n)
    gate = torch.full((size + 64,), 7, dtype=torch.uint8, device="cuda")
    out = torch.empty(m, n, dtype=torch.float16, device="cuda")
    f = _capi.LinearArgs(dtype=7, out_dtype=7, m=m, n=n, k=k, x=x.data_ptr(), weight=w.data_ptr(), out=out.data_ptr(), ld_x=k, ld_weight=k, ld_out=n,
                         act_type=act, act_alpha=LEAK, gate=gate.data_ptr())
    _capi.check(lib.cumm_hip_linear(ctypes.byref(f), stream))
    assert (gate[size:] == 7).all()
    got = []
    for kept in (gate, None):
        grads = [torch.full((r * c,), 7.0, device="cuda", dtype=torch.float16) for r, c in ((m, k), (n, k), (1, n))]
        a = _capi.LinearGradArgs(dtype=7, m=m, n=n, k=k, grad_out=dy.data_ptr(), x=x.data_ptr(), weight=w.data_ptr(), ld_grad_out=n, ld_x=k, ld_weight=k,
                                 grad_x=grads[0].data_ptr(), grad_weight=grads[1].data_ptr(), grad_bias=grads[2].data_ptr(), act_type=act, act_alpha=LEAK,
                                 from_inputs=1, gate=None if kept is None else kept.data_ptr())
        need = lib.cumm_hip_linear_backward_workspace(ctypes.byref(a))
        ws = torch.full((need + 512,), 7, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _capi.check(lib.cumm_hip_linear_backward(ctypes.byref(a), stream))
        assert (ws[need:] == 7).all()
        got.append(grads)
    assert all(torch.equal(a, b) for a, b in zip(*got))
    dz = torch.where(out > 0, STEP, STEP * (0.0 if act == 1 else LEAK)).double()
    assert torch.equal(got[0][0].view(m, k), R.mm(dz, w.double().t()).half())


def test_gates_of_a_captured_step(L):
    """Forward and backward in a graph, replayed with other numbers and with eager work in between."""
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda *shape: torch.randn(shape, generator=g, device="cuda").half()
    x, w, b, dy = new(700, 64).requires_grad_(), (new(128, 64) / 8).requires_grad_(), new(128).requires_grad_(), new(700, 128)

    def step():
        out = L.linear(x, w, b, activation="relu")
        grads = torch.autograd.grad(out, (x, w, b), dy)
        return (out.detach(),) + grads
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            x.copy_(new(700, 64))
            dy.copy_(new(700, 128))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, step()))
