"""What a saved-tensor hook gives back to the row-wise layers' backward passes: see test_layers_kept."""
import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

from test_layers_kept import spread

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["native", "python"])
def L(request):
    from cumm_amd import torch_bridge, torch_layers
    assert torch_bridge._native() is not None
    if request.param == "native":
        yield torch_layers
        return
    kept = torch_bridge._native_module
    torch_bridge._native_module = False
    yield torch_layers
    torch_bridge._native_module = kept


def steps(L):
    g = torch.Generator(device="cuda").manual_seed(3)
    new = lambda *shape: torch.randn(shape, generator=g, device="cuda").half().requires_grad_()
    x, w, b, r, wide, norm = new(2, 35, 24), new(40, 24), new(40), new(2, 35, 40), new(136, 24), new(24)
    return {
        "few channels": (lambda: L.linear(x, w, b, activation="silu", residual=r), (x, w, b), 3),
        "a gate": (lambda: L.linear(x, w, b, activation="relu", residual=r), (x, w, b), 3),
        "its argument": (lambda: L.linear(x, wide, activation="gelu"), (x, wide), 3),
        "its result": (lambda: L.linear(x, wide, activation="relu"), (x, wide), 3),
        "no activation": (lambda: L.linear(x, wide), (x, wide), 2),
        "norm": (lambda: L.rms_norm(x, norm), (x, norm), 3),
        "norm and sum": (lambda: sum(L.rms_norm(x, norm, residual=x)), (x, norm), 3),
    }


STEPS = ["few channels", "a gate", "its argument", "its result", "no activation", "norm", "norm and sum"]


def back(step, leaves, unpack):
    with saved_tensors_hooks(lambda t: t, unpack):
        out = step()
    return torch.autograd.grad(out, leaves, torch.ones_like(out))


@pytest.mark.parametrize("name", STEPS)
def test_other_strides(L, name):
    step, leaves, _ = steps(L)[name]
    want = back(step, leaves, lambda t: t)
    for unpack in (torch.clone, lambda t: spread(t) if t.dim() < 3 else torch.stack([spread(i) for i in t]), lambda t: t.flip(0).clone().flip(0),
                   lambda t: t.transpose(0, -1).contiguous().transpose(0, -1)):
        assert all(torch.equal(a, b) for a, b in zip(back(step, leaves, unpack), want))


@pytest.mark.parametrize("name", STEPS)
@pytest.mark.parametrize("what", ["type", "shape", "device"])
def test_others_are_refused(L, name, what):
    step, leaves, kept = steps(L)[name]
    for which in range(kept):
        seen = []

        def unpack(t):
            seen.append(t)
            if len(seen) - 1 != which:
                return t
            if what == "type":
                return t.float() if t.dtype != torch.float32 else t.half()
            return t[..., :-1] if what == "shape" else t.cpu()
        with pytest.raises(ValueError, match="came back"):
            back(step, leaves, unpack)
        assert len(seen) == kept
