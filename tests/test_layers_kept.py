"""What a saved-tensor hook gives back to the row-wise layers' backward passes, with a stand-in for the launch on the CPU: strides are
read, and a tensor that is not the kept one's like is refused before anything is launched."""
import contextlib

import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

from cumm_amd import torch_layers as L


@pytest.fixture
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(L, "_call", lambda fn, query, args, device: calls.append(args))
    monkeypatch.setattr(L, "_native", lambda: None)
    monkeypatch.setattr(L, "_on_device", lambda *a, **k: None)
    monkeypatch.setattr(L, "_Device", lambda device: contextlib.nullcontext())
    return calls


def layers():
    h = dict(dtype=torch.float16, requires_grad=True)
    x, w, b, r = torch.ones(6, 24, **h), torch.ones(40, 24, **h), torch.ones(40, **h), torch.ones(6, 40, **h)
    wide, norm = torch.ones(136, 24, **h), torch.ones(24, **h)
    return {
        "few channels": (lambda: L.linear(x, w, b, activation="silu", residual=r), 3),
        "a gate": (lambda: L.linear(x, w, b, activation="relu", residual=r), 3),
        "its argument": (lambda: L.linear(x, wide, activation="gelu"), 3),
        "its result": (lambda: L.linear(x, wide, activation="relu"), 3),
        "no activation": (lambda: L.linear(x, wide), 2),
        "norm": (lambda: L.rms_norm(x, norm), 3),
        "norm and sum": (lambda: L.rms_norm(x, norm, residual=x), 3),
    }


def back(layer, unpack):
    with saved_tensors_hooks(lambda t: t, unpack):
        out = layer()
    out = out if isinstance(out, tuple) else (out,)
    torch.autograd.backward(out, [torch.ones_like(t) for t in out])


def spread(t):
    """The same values, other strides"""
    if t.dim() == 1:
        return torch.stack((t, t), 1)[:, 0]
    field = torch.zeros(t.shape[0], t.shape[1] + 8, dtype=t.dtype, device=t.device)
    field[:, 3:3 + t.shape[1]] = t
    return field[:, 3:3 + t.shape[1]]


@pytest.mark.parametrize("name", layers())
def test_strides_are_read(launched, name):
    layer, _ = layers()[name]
    back(layer, spread)
    a = launched[-1]
    if name.startswith("norm"):
        assert a.ld_total == 24 + 8
    else:
        assert a.ld_weight == 24 + 8 and a.ld_x == 24 + 8
        if name.startswith("its"):
            assert a.ld_pre_act == 136 + 8


@pytest.mark.parametrize("name", layers())
@pytest.mark.parametrize("what", ["type", "shape", "device"])
def test_others_are_refused(launched, name, what):
    layer, kept = layers()[name]
    for which in range(kept):      # one of them at a time
        seen = []

        def unpack(t):
            seen.append(t)
            if len(seen) - 1 != which:
                return t
            if what == "type":
                return t.float() if t.dtype != torch.float32 else t.half()
            return t[..., :-1] if what == "shape" else t.to("meta")
        before = len(launched)
        with pytest.raises(ValueError, match="came back"):
            back(layer, unpack)
        assert len(launched) == before + 1 and len(seen) == kept      # the forward pass's
