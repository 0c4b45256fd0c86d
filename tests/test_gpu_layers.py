"""The row-wise layers (``cumm_amd.torch_layers``) against their formulas in 64 bits.

Bounds are derived, element by element: a rounding to a type is off by at most half a step, ``eps / 2`` of the value
(``EPS`` below); a sum of K products in 32 bits, in whatever order and whether an addition rounds or cuts, by at most
K 2^-23 of the sum of their magnitudes; an activation by its slope (at most 1.13) times the error of its argument plus
its own, 2^-21 of its argument (three hardware functions of one unit in the last place each and erf to 1.5e-7)."""
import math

import pytest
import torch

import layers_ref as R

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}      # half the smallest step
ACTS = ["none", "relu", "sigmoid", "leaky_relu", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def L():
    from cumm_amd import torch_bridge, torch_layers
    assert torch_bridge._native() is not None
    return torch_layers


@pytest.fixture(params=["native", "python"])
def either(request, L, monkeypatch):
    """The layers, and as a machine without a host compiler has them."""
    if request.param == "python":
        from cumm_amd import torch_bridge
        monkeypatch.setattr(torch_bridge, "_native_module", False)
    return L


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float16, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def within(got, want, allowed, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= allowed)
    if bad.any():
        i = bad.nonzero()[0]
        raise AssertionError("%s: %d of %d, first at %s: %g, want %g, allowed %g" % (
            what, int(bad.sum()), bad.numel(), i.tolist(), float(got[tuple(i)]), float(want[tuple(i)]), float(allowed[tuple(i)])))


def half_step(want, dtype):
    return want.abs() * EPS[dtype] + TINY[dtype]


def sum_error(a, b, terms):
    """of sums of products in 32 bits: a [m, k], b [n, k]"""
    return (terms + 8) * 2.0 ** -23 * R.mm(a.double().abs(), b.double().abs())


def linear_case(L, dtype, m, k, n, act, bias, residual, seed=0, pad=0, lead=0):
    """pad: rows lie that many elements further apart; lead: the first one begins that many elements behind a border"""
    g = gen(seed)

    def rows(r, c, scale=1.0):
        return normal(g, r * (c + pad) + lead, dtype=dtype, scale=scale)[lead:].view(r, c + pad)[:, :c]
    x, w = rows(m, k), rows(n, k, 1 / math.sqrt(k))
    b = normal(g, n + lead, dtype=dtype)[lead:] if bias else None
    r = rows(m, n) if residual else None
    got = L.linear(x, w, b, activation=act, residual=r, slope=0.2)
    assert got.shape == (m, n) and got.dtype == dtype and got.is_contiguous()
    z, want = R.linear(x, w, b, act, r, 0.2)
    err = sum_error(x, w, k) + z.abs() * 2.0 ** -23
    err = 1.13 * err + z.abs() * 2.0 ** -21 + want.abs() * 2.0 ** -23
    within(got, want, err * (1 + EPS[dtype]) + half_step(want, dtype), "linear")


SIZES = [  # m, k, n: one row and column to many tiles of every kernel; ends inside chunks of 16 bytes, steps, tiles
    (1, 1, 1), (1, 8, 8), (1, 4096, 40), (2, 7, 3), (3, 64, 17), (16, 512, 128), (17, 520, 136), (33, 129, 65), (64, 640, 1000),
    (65, 64, 64), (100, 72, 200), (127, 1000, 129), (128, 1024, 128), (200, 96, 1111), (256, 256, 256), (300, 1160, 776),
    (513, 2056, 264), (1000, 333, 520), (130, 8192, 96), (2049, 512, 2050), (5000, 32, 24), (777, 16, 9),
]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dtype", HALVES)
def test_linear_sizes(L, dtype, m, k, n):
    linear_case(L, dtype, m, k, n, "gelu", True, True, seed=m + k + n)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_linear_epilogues(L, act, bias, residual):
    for m, k, n in ((5, 96, 72), (150, 200, 264), (600, 128, 520)):
        linear_case(L, torch.bfloat16, m, k, n, act, bias, residual, seed=k)


@pytest.mark.parametrize("pad,lead", [(8, 0), (1, 0), (0, 1), (3, 5), (8, 4)])
@pytest.mark.parametrize("m,k,n", [(1, 64, 48), (40, 100, 33), (300, 256, 136)])
def test_linear_pitches_and_alignments(L, m, k, n, pad, lead):
    linear_case(L, torch.float16, m, k, n, "silu", True, True, seed=pad, pad=pad, lead=lead)


# rows at any address, read as they lie (in slices of k too) or copied: ends of rows in each place of a piece, of a step, one step
# after a slice; NaN around them
@pytest.mark.parametrize("m,k,n", [(1, 8, 5), (1, 9, 64), (6, 63, 70), (64, 65, 64), (70, 127, 130), (20, 129, 33), (5, 2299, 700), (300, 8191, 300), (17, 4097, 260),
                                   (2001, 191, 129), (3000, 193, 64), (16, 1025, 2050)])
@pytest.mark.parametrize("kind", HALVES + [torch.int8])
def test_linear_any_address(L, kind, m, k, n):
    for lead in (1, 2, 3, 6) if m < 100 else (3,):
        g = gen(lead)
        dtype = torch.float16 if kind == torch.int8 else kind

        def rows(r):
            if kind == torch.int8:      # what lies around the rows would be seen in every sum
                field = torch.full((r, k + 7), 127, device="cuda", dtype=torch.int8)
                field[:, lead:lead + k] = torch.randint(-127, 128, (r, k), generator=g, device="cuda").to(torch.int8)
            else:
                field = torch.full((r, k + 7), math.nan, device="cuda", dtype=dtype)
                field[:, lead:lead + k] = normal(g, r, k, dtype=dtype, scale=k ** -0.25)
            return field[:, lead:lead + k]
        x, w = rows(m), rows(n)
        if kind == torch.int8:
            xs, ws = torch.rand(m, generator=g, device="cuda") / 1000 + 1e-3, torch.rand(n, generator=g, device="cuda") / 1000 + 1e-3
            got = L.linear_s8(x, xs, w, ws, dtype=dtype)
            want = R.mm(x.double(), w.double()) * xs.double()[:, None] * ws.double()
            # the sum to 32 bits and two products of it
            within(got, want, want.abs() * 3 * 2.0 ** -24 * 1.01 + half_step(want, dtype) * 1.01, "linear_s8")
        else:
            b, r = normal(g, n, dtype=dtype), normal(g, m, n, dtype=dtype)
            got = L.linear(x, w, b, residual=r)
            _, want = R.linear(x, w, b, "none", r, 0)
            err = sum_error(x, w, k) + (want - r.double()).abs() * 2.0 ** -23 + want.abs() * 2.0 ** -23
            within(got, want, err * (1 + EPS[dtype]) + half_step(want, dtype), "linear")


# every tile in every layout, whole and in slices: large, 128 x 256, 128 x 128 in two and three stages, ends of k inside steps
@pytest.mark.parametrize("m,k,n", [(4093, 1000, 4088), (4093, 4088, 1000), (1000, 4088, 4093), (66000, 264, 680), (65272, 680, 168), (2040, 2056, 8200),
                                   (8200, 2040, 1030), (20000, 512, 520), (700, 20000, 500)])
def test_linear_large_sizes(L, m, k, n):
    check_gradients(L, "gelu" if k % 16 else "silu", torch.bfloat16 if m % 2 else torch.float16, m, k, n, m % 4 == 0)


def test_linear_large_tile(L):
    linear_case(L, torch.bfloat16, 4100, 1000, 4104, "gelu_tanh", True, True)
    linear_case(L, torch.float16, 4100, 520, 4001, "relu", True, False)


def test_linear_shapes_and_empty(either):
    L = either
    g = gen(1)
    x, w, b = normal(g, 2, 3, 5, 40), normal(g, 24, 40), normal(g, 24)
    got = L.linear(x, w, b)
    assert got.shape == (2, 3, 5, 24) and torch.equal(got.view(30, 24), L.linear(x.view(30, 40), w, b))
    assert torch.equal(L.linear(x.transpose(0, 1), w, b), got.transpose(0, 1))
    wide = normal(g, 2, 3, 5, 64)
    assert torch.equal(L.linear(wide[..., 8:48], w, b), L.linear(wide[..., 8:48].contiguous(), w, b))
    assert torch.equal(L.linear(wide[:, :2, 1:, 8:48], w, b), L.linear(wide[:, :2, 1:, 8:48].contiguous(), w, b))
    assert torch.equal(L.rms_norm(wide[..., 8:48], w[0]), L.rms_norm(wide[..., 8:48].contiguous(), w[0]))
    assert torch.equal(L.linear(x[1, 2, 3], w, b), L.linear(x[1, 2, 3:4], w, b)[0])
    assert L.linear(x[:0], w, b).shape == (0, 3, 5, 24)
    one = normal(g, 1, 1, 1, 24).expand(2, 3, 5, 24)
    assert torch.equal(L.linear(x, w, residual=one), L.linear(x, w, residual=one.contiguous()))
    assert torch.equal(L.linear(x, w.t().contiguous().t(), b), got)


def test_linear_not_numbers(L):
    """An infinity or a NaN reaches the rows and columns that have to do with it and no other; NaN passes every activation."""
    for m in (8, 300):
        x, w = normal(gen(2), m, 64), normal(gen(3), 48, 64)
        x[3, 5], x[5, 7] = float("nan"), float("inf")
        for act in ACTS:
            got = L.linear(x, w, activation=act)
            assert got[3].isnan().all(), act
            assert got[[i for i in range(m) if i not in (3, 5)]].isfinite().all(), act
        got = L.linear(x, w, activation="none")
        assert torch.equal(got[5], torch.where(w[:, 7] > 0, math.inf, -math.inf).half())


def test_linear_out_of_range_numbers_of_activations(L):
    """Arguments as large as the type has them: no NaN out of infinity times zero."""
    z = torch.tensor([-60000.0, -1000.0, -90.0, -20.0, -5.0, -1e-4, 0.0, 1e-4, 5.0, 20.0, 90.0, 1000.0, 60000.0], device="cuda").half()
    x, w = z.view(-1, 1), torch.ones(8, 1, device="cuda", dtype=torch.float16)
    for act in ACTS:
        got = L.linear(x, w, activation=act)
        _, want = R.linear(x, w, None, act, None, 0.01)
        assert got.isfinite().all(), act
        within(got, want, half_step(want, torch.float16) + 2.0 ** -21 * z.double().abs().view(-1, 1).clamp(max=20) + want.abs() * 2.0 ** -21, act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,k,n,residual", [(1, 8, 8, True), (3, 33, 17, False), (70, 64, 40, True), (300, 129, 264, False), (2000, 64, 128, True),
                                            (150, 2048, 200, False)])
def test_linear_gradients(L, act, dtype, m, k, n, residual):
    check_gradients(L, act, dtype, m, k, n, residual)


def check_gradients(L, act, dtype, m, k, n, residual):
    """The result and all gradients of a call against the formulas."""
    g = gen(m + n)
    x, w, b = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=1 / math.sqrt(k)), normal(g, n, dtype=dtype)
    r = normal(g, m, n, dtype=dtype) if residual else None
    dy = normal(g, m, n, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
    out = L.linear(x, w, b, activation=act, residual=r, slope=0.2)
    got = torch.autograd.grad(out, leaves, dy)
    with torch.no_grad():
        assert torch.equal(out, L.linear(x, w, b, activation=act, residual=r, slope=0.2))
        z, want = R.linear(x, w, b, act, r, 0.2)
        err = 1.13 * (sum_error(x, w, k) + z.abs() * 2.0 ** -23) + z.abs() * 2.0 ** -21 + want.abs() * 2.0 ** -23
        within(out, want, err * (1 + EPS[dtype]) + half_step(want, dtype), "linear")
        dz = dy.double() * R.slope(z, act, 0.2)
        # the argument is off by the sum's error and its rounding, the slope by at most 1.2 times that (its own
        # slope: 0.8 for the gelus, 0.5 for silu, 0.1 for the logistic function) and 2^-20; a kink may go either way
        off = sum_error(x, w, k) + half_step(z, dtype)
        at_kink = (z.abs() <= off) if act in ("relu", "leaky_relu") else torch.zeros_like(z, dtype=torch.bool)
        ddz = dy.double().abs() * (1.2 * off * (act not in ("none", "relu", "leaky_relu")) + 2.0 ** -20 + at_kink.double())
        sure = ddz                                   # of the unrounded dz
        ddz = ddz + (0 if act == "none" else 1) * half_step(dz, dtype)
        ax, aw = x.detach().double().abs(), w.detach().double().abs()
        tops = [R.mm(dz, w.detach().double().t()), R.mm(dz.t(), x.detach().double().t()), dz.sum(0)]
        mag = dz.abs() + ddz
        errs = [R.mm(ddz, aw.t()) + (n + 8) * 2.0 ** -23 * R.mm(mag, aw.t()), R.mm(ddz.t(), ax.t()) + (m + 8) * 2.0 ** -23 * R.mm(mag.t(), ax.t()),
                sure.sum(0) + (m + 8) * 2.0 ** -23 * mag.sum(0)]
        for name, a, want, err in zip(("grad_x", "grad_weight", "grad_bias"), got, tops, errs):
            assert a.dtype == dtype
            within(a, want, err * (1 + EPS[dtype]) + half_step(want, dtype), name)
        if residual:
            assert torch.equal(got[3], dy)


# few channels: one pass over the rows; a row, part of a wave's and of a workgroup's, several rounds of every workgroup
NARROW = [(1, 8, 8), (15, 64, 128), (16, 128, 64), (17, 72, 120), (127, 64, 64), (128, 128, 128), (129, 8, 128), (300, 128, 8), (1000, 40, 56),
          (32773, 24, 48), (70000, 128, 128), (70001, 64, 128), (33000, 128, 40)]


@pytest.mark.parametrize("m,k,n", NARROW)
@pytest.mark.parametrize("dtype", HALVES)
def test_narrow_gradients(L, dtype, m, k, n):
    for act in ACTS if m < 2000 else ("none", "relu", "gelu"):
        check_gradients(L, act, dtype, m, k, n, m % 2 == 0)


def test_narrow_pitches_and_alignments(either):
    L = either
    for lead, pad in ((0, 8), (1, 0), (3, 5), (8, 1)):
        g = gen(pad)
        rows = lambda r, c: normal(g, r * (c + pad) + lead)[lead:].view(r, c + pad)[:, :c]
        x, w, b, dy = rows(400, 64), rows(104, 64), normal(g, 104 + lead)[lead:], rows(400, 104)
        grads = lambda *t: torch.autograd.grad(L.linear(*t[:3], activation="silu"), t[:3], t[3])
        want = grads(*[t.contiguous().clone().requires_grad_(i < 3) for i, t in enumerate((x, w, b, dy))])
        got = grads(*[t.detach().requires_grad_(i < 3) for i, t in enumerate((x, w, b, dy))])
        assert all(torch.equal(a, c) for a, c in zip(got, want)), (lead, pad)


def test_narrow_not_numbers(L):
    """An infinite weight whose products are positive: ReLU passes it, and what does not have to do with it stays finite -
    the rows behind the last one are no rows, the channels behind the last one none either."""
    g = gen(4)
    for m, k, n in ((5, 64, 64), (131, 40, 24)):
        x, w, dy = normal(g, m, k).abs(), normal(g, n, k), normal(g, m, n)
        with torch.no_grad():
            w[3, 7] = math.inf
        x, w = x.requires_grad_(), w.requires_grad_()
        b = torch.zeros(n, device="cuda", dtype=torch.float16, requires_grad=True)
        gx, gw, gb = torch.autograd.grad(L.linear(x, w, b, activation="relu"), (x, w, b), dy)
        assert gw.isfinite().all() and gb.isfinite().all()
        want = R.mm(dy[:, 3:4].double().t(), x.detach().double().t())[0]
        mag = R.mm(dy[:, 3:4].double().abs().t(), x.detach().double().t())[0]
        within(gw[3], want, (m + 8) * 2.0 ** -23 * mag * 1.01 + half_step(want, torch.float16), "grad_weight")
        assert gx[:, [i for i in range(k) if i != 7]].isfinite().all() and not gx[:, 7].isfinite().any()
        x2 = x.detach().clone()
        x2[2, 5] = math.nan
        x2.requires_grad_()
        gx, gw, gb = torch.autograd.grad(L.linear(x2, w.detach().nan_to_num(posinf=1.0).requires_grad_(), b, activation="gelu"), (x2, w, b), dy, allow_unused=True)[:3]
        assert gx[2].isnan().all() and gx[[i for i in range(m) if i != 2]].isfinite().all() and gb.isnan().all()


def test_narrow_beyond_two_gigabytes(L):
    """Rows whose ends lie beyond 2^32 bytes."""
    m, k, n = 36_000_000, 64, 64
    x, dy = (torch.zeros(m, k, device="cuda", dtype=torch.float16) for _ in range(2))
    x[-300:], dy[-300:] = normal(gen(1), 300, k), normal(gen(2), 300, n)
    w = normal(gen(3), n, k, scale=1 / 8)
    leaves = [t.requires_grad_() for t in (x, w)]
    gx, gw = torch.autograd.grad(L.linear(x, w, activation="silu"), leaves, dy)
    with torch.no_grad():
        tail, d = x[-300:].double(), dy[-300:].double()
        dz = d * R.slope(R.mm(tail, w.double()), "silu", 0)
        # the slope's error: that of the argument's sum and 2^-20; dz rounded; the sum of the products
        ddz = d.abs() * (1.2 * sum_error(tail, w, k) + 2.0 ** -20) + half_step(dz, torch.float16)
        mag = dz.abs() + ddz
        want, aw = R.mm(dz, w.double().t()), w.double().abs().t()
        within(gx[-300:], want, (R.mm(ddz, aw) + (n + 8) * 2.0 ** -23 * R.mm(mag, aw)) * (1 + EPS[torch.float16]) + half_step(want, torch.float16), "grad_x")
        assert (gx[:-300] == 0).all()
        want, ax = R.mm(dz.t(), tail.t()), tail.abs().t()
        within(gw, want, (R.mm(ddz.t(), ax) + (300 + 8) * 2.0 ** -23 * R.mm(mag.t(), ax)) * (1 + EPS[torch.float16]) + half_step(want, torch.float16), "grad_weight")


def test_narrow_writes_its_results_only(L):
    import ctypes
    from cumm_amd import _capi
    g = gen(7)
    for m, k, n in ((3, 40, 24), (129, 64, 72), (300, 128, 8)):
        x, w, b, dy = normal(g, m, k), normal(g, n, k), normal(g, n), normal(g, m, n)
        fields = [torch.full((size + 40,), 7.0, device="cuda", dtype=torch.float16) for size in (m * k, n * k, n)]
        inner = [f[20:-20] for f in fields]
        a = _capi.LinearGradArgs(dtype=7, m=m, n=n, k=k, grad_out=dy.data_ptr(), x=x.data_ptr(), weight=w.data_ptr(), bias=b.data_ptr(), ld_grad_out=n, ld_x=k,
                                 ld_weight=k, grad_x=inner[0].data_ptr(), grad_weight=inner[1].data_ptr(), grad_bias=inner[2].data_ptr(), act_type=5, from_inputs=1)
        need = _capi.lib().cumm_hip_linear_backward_workspace(ctypes.byref(a))
        ws = torch.full((need + 512,), 7, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _capi.check(_capi.lib().cumm_hip_linear_backward(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
        leaves = [t.requires_grad_() for t in (x, w, b)]
        want = torch.autograd.grad(L.linear(*leaves, activation="gelu"), leaves, dy)
        assert all(torch.equal(i.view_as(t), t) for i, t in zip(inner, want)) and (ws[need:] == 7).all()
        for f, i in zip(fields, inner):
            i.fill_(7.0)
            assert (f == 7.0).all()


def test_narrow_layers_keep_their_operands(either):
    """What the activation got is worked out from the operands: one that was changed since is an error, as it is for any layer
    that keeps an operand."""
    L = either
    for changed in ("x", "w", "b"):
        t = dict(x=normal(gen(1), 40, 64).requires_grad_(), w=normal(gen(2), 32, 64), b=normal(gen(3), 32))
        leaf = t["x"]
        t["x"] = t["x"] * 1
        out = L.linear(t["x"], t["w"], t["b"], activation="silu")
        t[changed].add_(1)
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(out, leaf, torch.ones_like(out))


@pytest.mark.parametrize("wanted", ["x", "w", "b", "xw", "wb", "xb"])
@pytest.mark.parametrize("m,k,n", [(90, 40, 56), (200, 64, 128), (40, 200, 60)])
def test_some_gradients_without_an_activation(either, wanted, m, k, n):
    """Nothing is worked out again: an operand that no wanted gradient needs is not kept, and may change."""
    L = either
    g = gen(5)
    t = dict(x=normal(g, m, k), w=normal(g, n, k), b=normal(g, n))
    dy = normal(g, m, n)

    def grads(names, change=()):
        leaves = {k: v.detach().clone().requires_grad_(k in names) for k, v in t.items()}
        out = L.linear(leaves["x"], leaves["w"], leaves["b"])
        for name in change:
            leaves[name].add_(1)
        return dict(zip(names, torch.autograd.grad(out, [leaves[k] for k in names], dy)))
    all_of_them = grads("xwb")
    some = grads(wanted, "xw" if wanted == "b" else "")
    for name in wanted:
        assert torch.equal(some[name], all_of_them[name]), name


def test_the_same_tensor_twice(either):
    """x as its own residual, as its own weight, and under a norm as its own residual: the gradients add up."""
    L = either
    for c, act in ((64, "silu"), (200, "gelu")):
        x, dy, w = normal(gen(1), c, c, scale=0.5), normal(gen(2), c, c), normal(gen(3), c, c, scale=c ** -0.5)
        n = normal(gen(4), c)
        one, two = x.clone().requires_grad_(), [x.clone().requires_grad_() for _ in range(2)]
        got, = torch.autograd.grad(L.linear(one, w, activation=act, residual=one), one, dy)
        parts = torch.autograd.grad(L.linear(two[0], w, activation=act, residual=two[1]), two, dy)
        assert torch.equal(got, parts[0] + parts[1])
        got, = torch.autograd.grad(L.linear(one, one, activation=act), one, dy)
        parts = torch.autograd.grad(L.linear(two[0], two[1], activation=act), two, dy)
        assert torch.equal(got, parts[0] + parts[1])
        got, = torch.autograd.grad(L.rms_norm(one, n, residual=one), one, (dy, dy))
        parts = torch.autograd.grad(L.rms_norm(two[0], n, residual=two[1]), two, (dy, dy))
        assert torch.equal(got, parts[0] + parts[1])


@pytest.mark.parametrize("wanted", ["x", "w", "b", "xw", "wb", "xb"])
def test_wide_some_gradients(either, wanted):
    L = either
    g = gen(5)
    t = dict(x=normal(g, 90, 200), w=normal(g, 60, 200), b=normal(g, 60))
    dy = normal(g, 90, 60)

    def grads(names):
        leaves = {k: v.detach().clone().requires_grad_(k in names) for k, v in t.items()}
        out = L.linear(leaves["x"], leaves["w"], leaves["b"], activation="gelu")
        return dict(zip(names, torch.autograd.grad(out, [leaves[k] for k in names], dy)))
    all_of_them, some = grads("xwb"), grads(wanted)
    for name in wanted:
        assert torch.equal(some[name], all_of_them[name]), name


@pytest.mark.parametrize("act", ["sigmoid", "leaky_relu", "silu", "gelu", "gelu_tanh"])
def test_linear_gradient_against_differences(L, act):
    """The slope that the backward pass uses, against differences of the formula in 64 bits."""
    z = torch.linspace(-7.9, 7.9, 401, device="cuda").bfloat16().unique().view(-1, 1)
    w = torch.ones(8, 1, device="cuda", dtype=torch.bfloat16)
    z.requires_grad_()
    got, = torch.autograd.grad(L.linear(z, w, activation=act, slope=0.25), z, torch.ones(z.shape[0], 8, device="cuda", dtype=torch.bfloat16))
    d, step = z.detach().double(), 1e-5
    want = 8 * (R.act(d + step, act, 0.25) - R.act(d - step, act, 0.25)) / (2 * step)
    far = d.abs() > 1e-3 if act == "leaky_relu" else torch.ones_like(d, dtype=torch.bool)
    # eight slopes, each rounded once, added and rounded again; differences are off by less than step^2
    within(torch.where(far, got, 0), torch.where(far, want, 0.0), 2 * half_step(want, torch.bfloat16) + 8 * 2.0 ** -19, act)


@pytest.mark.parametrize("wanted", ["x", "w", "b", "r", "xw", "wb", "xb"])
def test_linear_some_gradients(either, wanted):
    L = either
    g = gen(5)
    t = dict(x=normal(g, 90, 40), w=normal(g, 56, 40), b=normal(g, 56), r=normal(g, 90, 56))
    dy = normal(g, 90, 56)

    def grads(names):
        leaves = {k: v.detach().clone().requires_grad_(k in names) for k, v in t.items()}
        out = L.linear(leaves["x"], leaves["w"], leaves["b"], activation="gelu", residual=leaves["r"])
        return dict(zip(names, torch.autograd.grad(out, [leaves[k] for k in names], dy)))
    all_of_them, some = grads("xwbr"), grads(wanted)
    for name in wanted:
        assert torch.equal(some[name], all_of_them[name]), name


def test_linear_gradient_of_strided_and_broadcast_results(either):
    """A gradient that is a number spread out, or a transposed view; leading dimensions; no rows at all."""
    L = either
    g = gen(6)
    x, w, b = (t.requires_grad_() for t in (normal(g, 4, 9, 40), normal(g, 24, 40), normal(g, 24)))
    dy = normal(g, 9, 24, 4).permute(2, 0, 1)
    got = torch.autograd.grad(L.linear(x, w, b, activation="silu"), (x, w, b), dy)
    want = torch.autograd.grad(L.linear(x, w, b, activation="silu"), (x, w, b), dy.contiguous())
    assert all(torch.equal(a, c) for a, c in zip(got, want)) and got[0].shape == x.shape
    one = torch.ones((), device="cuda", dtype=torch.float16).expand(4, 9, 24)
    got = torch.autograd.grad(L.linear(x, w, b), (x, w, b), one)
    assert torch.equal(got[2], torch.full((24,), 36.0, device="cuda").half())
    got = torch.autograd.grad(L.linear(x[:0], w, b, activation="gelu"), (w, b), dy[:0])
    assert all((t == 0).all() for t in got)
    with pytest.raises(RuntimeError):      # once differentiable
        first, = torch.autograd.grad(L.linear(x, w, b, activation="silu").float().square().sum(), x, create_graph=True)
        torch.autograd.grad(first.float().sum(), w)


S8_SIZES = [(4093, 4096, 4100), (300, 16384, 300), (1100, 8192, 4096), (60000, 64, 70), (1, 1, 1), (1, 4096, 100), (5, 17, 33), (16, 1024, 256), (40, 80, 24), (64, 4096, 520), (65, 128, 64), (130, 4100, 132), (500, 1003, 777), (2000, 512, 520)]


@pytest.mark.parametrize("m,k,n", S8_SIZES)
@pytest.mark.parametrize("dtype", HALVES)
def test_linear_s8(L, dtype, m, k, n):
    g = gen(m * k + n)
    x = torch.randint(-128, 128, (m, k), generator=g, device="cuda").to(torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda").to(torch.int8)
    xs, ws = torch.rand(m, generator=g, device="cuda") / 100, torch.rand(n, generator=g, device="cuda") / (100 * math.sqrt(k))
    b, r = torch.randn(n, generator=g, device="cuda"), normal(g, m, n, dtype=dtype)
    got = L.linear_s8(x, xs, w, ws, b, activation="silu", residual=r, dtype=dtype)
    exact = R.mm(x.double(), w.double())
    z = exact * xs.double()[:, None] * ws.double() + b.double()
    want = R.act(z, "silu", 0) + r.double()
    # the sum is exact, its conversion, two products and an addition are rounded once each
    err = 4 * 2.0 ** -24 * ((exact * xs.double()[:, None] * ws.double()).abs() + b.double().abs())
    err = 1.13 * err + z.abs() * 2.0 ** -21 + want.abs() * 2.0 ** -23
    within(got, want, err * (1 + EPS[dtype]) + half_step(want, dtype), "linear_s8")


def test_linear_s8_sums_are_whole_numbers(L):
    """The largest sums that there may be."""
    x = torch.full((3, 131071), -128, device="cuda", dtype=torch.int8)
    w = torch.full((8, 131071), -128, device="cuda", dtype=torch.int8)
    w[1] = 127
    one = torch.ones(8, device="cuda")
    got = L.linear_s8(x, one[:3] * 2.0 ** -20, w, one * 2.0 ** -4, dtype=torch.bfloat16)
    want = torch.tensor([131071 * 128.0 * 128, -131071 * 128.0 * 127], dtype=torch.float64) / 2 ** 24
    assert torch.equal(got[:, :2].cpu(), want.to(torch.bfloat16).expand(3, 2))


NORM_SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (9, 100), (4, 512), (7, 513), (5, 1024), (6, 1025), (3, 2048), (4, 2056), (130, 4096), (9, 5000), (17, 8192),
              (3, 8200), (2, 16384), (5, 16392), (2, 20001), (3, 32768), (2, 32776), (3, 70001), (1000, 40), (3001, 256)]


def norm_rows(g, m, k, dtype, pad=0, lead=0):
    t = torch.randn((m, k + pad), generator=g, device="cuda") * torch.exp(torch.randn((m, 1), generator=g, device="cuda"))
    flat = torch.empty(m * (k + pad) + lead, dtype=dtype, device="cuda")
    flat[lead:].view(m, k + pad).copy_(t)
    return flat[lead:].view(m, k + pad)[:, :k]


def check_norm(L, dtype, x, r, w, eps=1e-5):
    m, k = x.shape
    got = L.rms_norm(x, w, eps, residual=r)
    s8 = L.rms_norm_s8(x, w, eps, residual=r)
    h = x.double()
    if r is not None:
        assert torch.equal(got[1], x + r) and torch.equal(s8[2], got[1])
        h, got = got[1].double(), got[0]
    inv = 1 / (h.square().mean(1, keepdim=True) + eps).sqrt()
    want = h * inv * w.double()
    # the mean of squares: k + 8 roundings of 2^-24 of a sum of positive numbers, halved by the root; root, quotient and
    # products a rounding each
    rel = ((k + 8) * 2.0 ** -25 + 6 * 2.0 ** -24)
    within(got, want, want.abs() * rel * (1 + EPS[dtype]) + half_step(want, dtype), "rms_norm")
    # 127 v / top for v exact in 32 bits: codes are whole numbers without a tolerance
    v = (h.float() * w.float()).double()
    top = v.abs().amax(1, keepdim=True)
    codes = torch.where(top > 0, torch.round(v * 127 / top.clamp_min(1e-300)), 0.0)
    assert torch.equal(s8[0].double(), codes)
    scale = (top * inv / 127)[:, 0]
    within(s8[1], scale, scale * (rel + 2.0 ** -23) + 2.0 ** -149, "scale")


@pytest.mark.parametrize("m,k", NORM_SIZES)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_sizes(L, dtype, m, k, residual):
    g = gen(m + k)
    check_norm(L, dtype, norm_rows(g, m, k, dtype), norm_rows(g, m, k, dtype) if residual else None, normal(g, k, dtype=dtype, scale=0.3) + 1)


@pytest.mark.parametrize("pad,lead", [(1, 0), (0, 3), (8, 0), (5, 1)])
@pytest.mark.parametrize("k", [40, 1001, 2048])
def test_norm_pitches_and_alignments(L, k, pad, lead):
    g = gen(k + pad)
    x, r = norm_rows(g, 11, k, torch.bfloat16, pad, lead), norm_rows(g, 11, k, torch.bfloat16, pad + 2, lead)
    check_norm(L, torch.bfloat16, x, r, normal(g, k + lead, dtype=torch.bfloat16)[lead:])


@pytest.mark.parametrize("dtype", HALVES + [torch.float32])
@pytest.mark.parametrize("m,k", NORM_SIZES)
def test_quantize_rows(L, dtype, m, k):
    g = gen(m * 3 + k)
    x = torch.randn((m, k), generator=g, device="cuda").to(dtype)
    codes, scale = L.quantize_rows(x)
    top = x.double().abs().amax(1, keepdim=True)
    assert torch.equal(codes.double(), torch.round(x.double() * 127 / top))
    assert int(codes.abs().max()) == 127
    within(scale, (top / 127)[:, 0], (top / 127)[:, 0] * 2.0 ** -24, "scale")


def test_quantize_ties_and_extremes(L):
    """Quotients that are ties exactly (to even), one step of 32 bits beside them, and tiny and huge rows."""
    ties = torch.arange(-126, 127, device="cuda").float() + 0.5
    for top in (127.0, 127.0 * 2 ** -20, 254.0, 127.0 * 3, 127.0 * 2.0 ** 100, 127.0 * 2.0 ** -140):
        at = ties[(ties.abs() < 127)] * (top / 127)
        row = torch.cat([torch.tensor([top], device="cuda"), at, torch.nextafter(at, at + at.abs() + 1e-30), torch.nextafter(at, at - at.abs() - 1e-30)])
        codes, scale = L.quantize_rows(row.view(1, -1))
        want = torch.round(row.double() * 127 / row.double().abs().max())
        assert torch.equal(codes[0].double(), want), top
    x = torch.zeros(5, 100, device="cuda")
    x[1, 3], x[2, 4], x[3, :], x[4, 0] = float("inf"), float("nan"), 1.0, 3e38
    x[1, 5] = 2.0
    codes, scale = L.quantize_rows(x)
    assert (codes[:3] == 0).all() and scale[0] == 0 and scale[1] == float("inf") and scale[2].isnan()
    assert (codes[3] == 127).all() and codes[4, 0] == 127 and (codes[4, 1:] == 0).all()
    q = L.quantize_rows(x[3:4].view(2, 50)[:, :0 + 50].half())
    assert q[0].shape == (2, 50) and q[1].shape == (2,)
    assert L.quantize_rows(x[:0])[0].shape == (0, 100)


def test_norm_rows_of_zeros_and_not_numbers(L):
    x = normal(gen(3), 6, 200, dtype=torch.bfloat16)
    w = torch.ones(200, device="cuda", dtype=torch.bfloat16)
    x[0], x[2, 7], x[4, 9] = 0, float("nan"), float("inf")
    out = L.rms_norm(x, w)
    assert (out[0] == 0).all() and out[2].isnan().all() and out[4, 9].isnan() and (out[4, :9] == 0).all()
    assert out[[1, 3, 5]].isfinite().all()
    codes, scale = L.rms_norm_s8(x, w)
    assert (codes[[0, 2, 4]] == 0).all() and scale[0] == 0 and not scale[[2, 4]].isfinite().any()
    assert scale[[1, 3, 5]].isfinite().all()


@pytest.mark.parametrize("m,k", [(1, 8), (3, 7), (50, 64), (33, 512), (40, 1001), (70, 2048), (600, 300), (9, 4096), (21, 8192), (5, 12000), (3, 16384), (7, 20001), (5000, 96)])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_gradients(L, dtype, m, k, residual):
    g = gen(m + 2 * k)
    x, w = normal(g, m, k, dtype=dtype).requires_grad_(), (normal(g, k, dtype=dtype, scale=0.3) + 1).requires_grad_()
    r = normal(g, m, k, dtype=dtype).requires_grad_() if residual else None
    dy, ds = normal(g, m, k, dtype=dtype), normal(g, m, k, dtype=dtype)
    out = L.rms_norm(x, w, 1e-5, residual=r)
    leaves = [x, w] + ([r] if residual else [])
    got = torch.autograd.grad(out, leaves, (dy, ds) if residual else dy)
    with torch.no_grad():
        plain = L.rms_norm(x, w, 1e-5, residual=r)
        assert torch.equal(out[0], plain[0]) and torch.equal(out[1], plain[1]) if residual else torch.equal(out, plain)
        h = out[1].double() if residual else x.double()
        inv = 1 / (h.square().mean(1, keepdim=True) + 1e-5).sqrt()
        u, gw = h * inv, dy.double() * w.double()
        dot = (gw * u).mean(1, keepdim=True)
        dh = inv * (gw - u * dot) + (ds.double() if residual else 0)
        rel = (k + 8) * 2.0 ** -25 + 8 * 2.0 ** -24
        size = inv * (gw.abs() + u.abs() * (gw * u).abs().mean(1, keepdim=True))
        err = size * (2 * rel + (k + 8) * 2.0 ** -24) + dh.abs() * 2.0 ** -23
        within(got[0], dh, err * (1 + EPS[dtype]) + half_step(dh, dtype), "grad_x")
        dw = (dy.double() * u).sum(0)
        err = (dy.double() * u).abs().sum(0) * (rel + (m + 8) * 2.0 ** -24)
        within(got[1], dw, err * (1 + EPS[dtype]) + half_step(dw, dtype), "grad_weight")
        if residual:
            assert torch.equal(got[2], got[0])


def test_norm_gradient_against_differences(L):
    x, w = normal(gen(8), 2, 24, dtype=torch.float16), normal(gen(9), 24, dtype=torch.float16) + 1
    x.requires_grad_()
    dy = normal(gen(10), 2, 24)
    got, = torch.autograd.grad(L.rms_norm(x, w, 1e-3), x, dy)
    f = lambda h: (h / (h.square().mean(1, keepdim=True) + 1e-3).sqrt() * w.double() * dy.double()).sum()
    d, step = x.detach().double(), 1e-5
    for i in range(2):
        for j in range(24):
            e = torch.zeros_like(d)
            e[i, j] = step
            want = (f(d + e) - f(d - e)) / (2 * step)
            assert abs(float(got[i, j]) - float(want)) <= abs(float(want)) * EPS[torch.float16] + 1e-5


def test_norm_gradients_of_one_result_only(either):
    """A gradient of the sum alone, or of the norm alone, or with parts that want none."""
    L = either
    g = gen(4)
    x, r, w = (normal(g, 12, 72).requires_grad_(), normal(g, 12, 72).requires_grad_(), normal(g, 72).requires_grad_())
    dy = normal(g, 12, 72)
    out, total = L.rms_norm(x, w, residual=r)
    got = torch.autograd.grad(total, (x, r, w), dy, allow_unused=True, retain_graph=True)
    assert torch.equal(got[0], dy) and torch.equal(got[1], dy) and (got[2] is None or (got[2] == 0).all())
    zero = torch.autograd.grad((out, total), (x, w), (dy, torch.zeros_like(dy)), retain_graph=True)
    alone = torch.autograd.grad(out, (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(alone, zero))
    frozen = L.rms_norm(x, w.detach(), residual=r.detach())[0]
    assert torch.equal(torch.autograd.grad(frozen, x, dy)[0], alone[0])
    only_w = L.rms_norm(x.detach(), w, residual=r.detach())[0]
    assert torch.equal(torch.autograd.grad(only_w, w, dy)[0], alone[1])
    empty = L.rms_norm(x[:0], w, residual=r[:0])[0]
    assert (torch.autograd.grad(empty, w, dy[:0])[0] == 0).all()


def test_same_bits_from_run_to_run(either):
    L = either
    g = gen(11)
    x, w, b = (t.requires_grad_() for t in (normal(g, 3000, 96), normal(g, 136, 96), normal(g, 136)))
    n = normal(g, 96).requires_grad_()
    dy = normal(g, 3000, 136)

    def once():
        out = L.linear(L.rms_norm(x, n), w, b, activation="silu")
        return (out.detach(),) + torch.autograd.grad(out, (x, w, b, n), dy)
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, once()))


def block(L, x, skip, p):
    """A feed-forward block as inference runs it in 8 bits: norm, widening product, narrowing product, the residual stream."""
    codes, scale, skip = L.rms_norm_s8(x, p["norm"], residual=skip)
    wide = L.linear_s8(codes, scale, p["up"], p["up_scale"], p["up_bias"], activation="gelu", dtype=x.dtype)
    codes, scale = L.quantize_rows(wide)
    return L.linear_s8(codes, scale, p["down"], p["down_scale"], residual=skip, dtype=x.dtype), skip


def block_weights(L, g, k, dtype):
    up, down = normal(g, 4 * k, k, dtype=torch.float32, scale=k ** -0.5), normal(g, k, 4 * k, dtype=torch.float32, scale=(4 * k) ** -0.5)
    p = dict(norm=torch.ones(k, device="cuda", dtype=dtype), up_bias=normal(g, 4 * k, dtype=torch.float32, scale=0.1), full=(up, down))
    p["up"], p["up_scale"] = L.quantize_rows(up)
    p["down"], p["down_scale"] = L.quantize_rows(down)
    return p


@pytest.mark.parametrize("m", [1, 7, 300])
@pytest.mark.parametrize("dtype", HALVES)
def test_block_in_8_bits(L, dtype, m):
    g = gen(m)
    k = 256
    p = block_weights(L, g, k, dtype)
    x, skip = normal(g, m, k, dtype=dtype), normal(g, m, k, dtype=dtype)
    got, total = block(L, x, skip, p)
    # the same steps in 64 bits out of the 8-bit numbers of each
    codes, scale, h = L.rms_norm_s8(x, p["norm"], residual=skip)
    wide = R.mm(codes.double() * scale.double()[:, None], p["up"].double() * p["up_scale"].double()[:, None]) + p["up_bias"].double()
    wide = R.act(wide, "gelu", 0).to(dtype)
    q, s = L.quantize_rows(wide)
    want = R.mm(q.double() * s.double()[:, None], p["down"].double() * p["down_scale"].double()[:, None]) + h.double()
    assert torch.equal(total, h)
    # two roundings of the wide row may differ by a step of the type, and its code by one: 1 / 254 of its largest value, in
    # half of the 4 k products at most, times a weight's largest value
    step = (s.double()[:, None] + wide.double().abs().amax(1, keepdim=True) * 2 * EPS[dtype]) * (p["down"].double() * p["down_scale"].double()[:, None]).abs().sum(1)
    within(got, want, step + half_step(want, dtype), "block")
    # and against the block without 8-bit numbers: a few in a hundred
    u, d = p["full"]
    hn = h.double() / (h.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
    full = R.mm(R.act(R.mm(hn, u.double()) + p["up_bias"].double(), "gelu", 0), d.double())
    assert float((got.double() - h.double() - full).norm() / full.norm()) < 0.05


def test_block_trains(either):
    """Norm, two products and the residual stream, forward and backward, against the formula's gradients in 64 bits."""
    L = either
    torch.manual_seed(0)
    norm, up, down = L.RMSNorm(96, dtype=torch.bfloat16), L.Linear(96, 200, activation="gelu_tanh", dtype=torch.bfloat16), L.Linear(200, 96, dtype=torch.bfloat16)
    x = torch.randn(3, 50, 96, device="cuda").bfloat16().requires_grad_()
    dy = torch.randn(3, 50, 96, device="cuda").bfloat16()
    params = [x] + list(norm.parameters()) + list(up.parameters()) + list(down.parameters())
    got = torch.autograd.grad(down(up(norm(x)), residual=x), params, dy)
    d = [t.detach().double().requires_grad_() for t in params]
    h = d[0] / (d[0].square().mean(-1, keepdim=True) + 1e-6).sqrt() * d[1]
    z = R.act((h.reshape(-1, 96) @ d[2].t().contiguous() + d[3]), "gelu_tanh", 0)
    want = torch.autograd.grad((z @ d[4].t().contiguous() + d[5]).view(3, 50, 96) + d[0], d, dy.double())
    for a, c in zip(got, want):
        # norm, wide row, its argument, dz twice and the result: six roundings of 2^-9 on average
        assert float((a.double() - c).norm() / c.norm()) < 6 * 2.0 ** -8


def replays(run, static, eager):
    """Captured once, replayed with new values in the same memory, the program's own calls in between."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = run()
    for i in range(4):
        for t in static:
            with torch.no_grad():
                t.copy_(normal(gen(100 + i), *t.shape, dtype=t.dtype))
        want = eager()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


@pytest.mark.parametrize("m", [1, 40, 700])
def test_captured_inference(L, m):
    g = gen(m)
    p = block_weights(L, g, 128, torch.float16)
    x, skip = normal(g, m, 128), normal(g, m, 128)
    run = lambda: block(L, x, skip, p)
    replays(run, [x, skip], run)


def test_captured_training_step(either):
    """Forward and backward of the same leaves in one graph; eager passes take leaves of their own."""
    L = either
    g = gen(2)
    shapes = [(200, 72), (72,), (130, 72), (130,), (200, 130)]
    t = [normal(g, *s).requires_grad_() for s in shapes[:4]] + [normal(g, *shapes[4])]

    def step(x, n, w, b, dy):
        out = L.linear(L.rms_norm(x, n), w, b, activation="gelu")
        return (out.detach(),) + torch.autograd.grad(out, (x, n, w, b), dy)
    eager = lambda: step(*[v.detach().clone().requires_grad_(v.requires_grad) for v in t])
    replays(lambda: step(*t), t, eager)


def test_captured_narrow_training_step(either):
    L = either
    g = gen(2)
    t = [normal(g, *s).requires_grad_() for s in ((700, 72), (104, 72), (104,))] + [normal(g, 700, 104)]

    def step(x, w, b, dy):
        out = L.linear(x, w, b, activation="gelu")
        return (out.detach(),) + torch.autograd.grad(out, (x, w, b), dy)
    eager = lambda: step(*[v.detach().clone().requires_grad_(v.requires_grad) for v in t])
    replays(lambda: step(*t), t, eager)


def test_two_streams_at_once(L):
    """Calls on two streams, each with a workspace of its own, while both run."""
    g = gen(3)
    x, w = normal(g, 300, 4096), normal(g, 264, 4096, scale=1 / 64)
    want = L.linear(x, w, activation="silu")
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(L.linear(x, w, activation="silu"))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) for a in got)


def test_behind_the_last_row_nothing_is_written(L):
    """The rows and columns around the result's, by the C entry points, which take pitches and places."""
    import ctypes
    from cumm_amd import _capi
    g = gen(7)
    for m, k, n in ((3, 40, 21), (70, 64, 72), (300, 128, 200)):
        x, w, r = normal(g, m, k), normal(g, n, k), normal(g, m, n)
        field = torch.full((m + 2, n + 9), 7.0, device="cuda", dtype=torch.float16)
        pre = torch.full((m + 2, n + 5), 7.0, device="cuda", dtype=torch.float16)
        inner, inner_pre = field[1:-1, 4:4 + n], pre[1:-1, 2:2 + n]
        a = _capi.LinearArgs(dtype=7, out_dtype=7, m=m, n=n, k=k, x=x.data_ptr(), weight=w.data_ptr(), residual=r.data_ptr(), out=inner.data_ptr(),
                             pre_act=inner_pre.data_ptr(), ld_x=k, ld_weight=k, ld_residual=n, ld_out=n + 9, ld_pre_act=n + 5, act_type=4)
        need = _capi.lib().cumm_hip_linear_workspace(ctypes.byref(a))
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        _capi.check(_capi.lib().cumm_hip_linear(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
        assert torch.equal(inner, L.linear(x, w, activation="silu", residual=r))
        assert torch.equal(inner_pre, L.linear(x, w))
        for t, i in ((field, inner), (pre, inner_pre)):
            i.fill_(7.0)
            assert (t == 7.0).all()


def test_result_over_the_residual(L):
    import ctypes
    from cumm_amd import _capi
    for m, k, n in ((4, 64, 40), (90, 4096, 72), (500, 96, 264)):
        x, w, r = normal(gen(m), m, k), normal(gen(n), n, k, scale=k ** -0.5), normal(gen(k), m, n)
        want = L.linear(x, w, residual=r, activation="relu")
        a = _capi.LinearArgs(dtype=7, out_dtype=7, m=m, n=n, k=k, x=x.data_ptr(), weight=w.data_ptr(), residual=r.data_ptr(), out=r.data_ptr(), ld_x=k,
                             ld_weight=k, ld_residual=n, ld_out=n, act_type=1)
        ws = torch.empty(max(_capi.lib().cumm_hip_linear_workspace(ctypes.byref(a)), 1), dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        _capi.check(_capi.lib().cumm_hip_linear(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
        assert torch.equal(r, want)


def test_more_than_two_gigabytes(L):
    """Operands and results whose ends lie beyond 2^31 bytes, and beyond 2^32."""
    m, k = 600000, 2048
    x = torch.zeros(m, k, device="cuda", dtype=torch.float16)
    tail = normal(gen(1), 300, k)
    x[-300:] = tail
    w = normal(gen(2), 40, k, scale=1 / 32)
    got = L.linear(x, w)
    # (not the bits of a call with the last rows alone: fewer rows, another order of the sums - by the formula instead)
    _, want = R.linear(tail, w, None, "none", None, 0)
    within(got[-300:], want, sum_error(tail, w, k) * 1.01 + half_step(want, torch.float16), "linear")
    assert (got[:-300] == 0).all()
    dy = torch.ones(m, 40, device="cuda", dtype=torch.float16)
    wg = w.clone().requires_grad_()
    xs = x.detach()
    gw, = torch.autograd.grad(L.linear(xs, wg), wg, dy)
    want = tail.double().sum(0).expand(40, k)
    within(gw, want, (300 + 8) * 2.0 ** -23 * tail.double().abs().sum(0).expand(40, k) + half_step(want, torch.float16) * 1.01, "grad_weight")
    n = torch.ones(k, device="cuda", dtype=torch.float16)
    assert torch.equal(L.rms_norm(x, n)[-300:], L.rms_norm(tail, n))
    codes, scale = L.quantize_rows(x)
    small = L.quantize_rows(tail)
    assert torch.equal(codes[-300:], small[0]) and torch.equal(scale[-300:], small[1])


@pytest.mark.parametrize("m,k,n", [(1, 64, 48), (33, 100, 40), (300, 256, 264)])
def test_both_halves_give_the_same(L, monkeypatch, m, k, n):
    from cumm_amd import torch_bridge
    g = gen(m)
    x, w, b, r, nw = (t.requires_grad_() for t in (normal(g, m, k), normal(g, n, k, scale=k ** -0.5), normal(g, n), normal(g, m, n), normal(g, k)))
    dy = normal(g, m, n)

    def all_of_it():
        h, total = L.rms_norm(x, nw, residual=x.detach())
        out = L.linear(h, w, b, activation="gelu", residual=r)
        grads = torch.autograd.grad((out, total), (x, w, b, r, nw), (dy, dy[:, :1].expand(m, k)))
        with torch.no_grad():
            codes = L.rms_norm_s8(x, nw, residual=x)
            q = L.quantize_rows(w)
            s8 = L.linear_s8(codes[0], codes[1], q[0], q[1], b.float(), activation="silu", residual=r, dtype=torch.float16)
        return (out, h, total, s8) + grads + codes + q
    native = all_of_it()
    monkeypatch.setattr(torch_bridge, "_native_module", False)
    own = all_of_it()
    assert len(native) == len(own) and all(torch.equal(a, c) and a.dtype == c.dtype for a, c in zip(native, own))
