"""Calls of the row-wise layers that somebody records or differentiates in forward mode: the launch goes past torch, so a record of
torch's operators alone would return memory that nobody wrote.  The launch here is a stand-in on the CPU."""
import contextlib
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from cumm_amd import torch_layers as L
from layers_calls import NAMES, calls

ONE = b"\x00\x3c"      # in f16


@pytest.fixture
def stand_in(monkeypatch):
    launched = []

    def call(fn, query, args, device):
        launched.append(args)
        m, n = args.m, getattr(args, "n", args.k)
        for at, size, value in ((getattr(args, "out", None), m * n, ONE), (getattr(args, "total", None), m * args.k, ONE),
                                (getattr(args, "codes", None), m * args.k, b"\x05"), (getattr(args, "scale", None), m, b"\x00\x00\x80\x3f")):
            if at:
                ctypes.memmove(at, value * size, len(value) * size)
    monkeypatch.setattr(L, "_call", call)
    monkeypatch.setattr(L, "_native", lambda: None)
    monkeypatch.setattr(L, "_on_device", lambda *a, **k: None)
    monkeypatch.setattr(L, "_Device", lambda device: contextlib.nullcontext())
    return launched


@pytest.mark.parametrize("name", NAMES)
def test_traces_hold_the_launch(stand_in, name):
    fn, tensors = calls(L, "cpu")[name]
    with torch.no_grad():
        traced = torch.jit.trace(fn, tensors, check_trace=False)
        assert "PythonOp" in str(traced.graph) or "^_" in str(traced.graph)
        before = len(stand_in)
        got = traced(*calls(L, "cpu", seed=1, rows=9)[name][1])
        assert len(stand_in) == before + 1 and all(t.shape[0] == 9 for t in got)
        want = fn(*calls(L, "cpu", seed=1, rows=9)[name][1])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("mode", ["real", "fake"])
def test_graphs_of_operators_are_refused(stand_in, name, mode):
    from torch.fx.experimental.proxy_tensor import make_fx
    fn, tensors = calls(L, "cpu")[name]
    with pytest.raises(ValueError, match="recorded"):
        make_fx(fn, tracing_mode=mode)(*tensors)
    assert not stand_in
    assert fn(*tensors) and len(stand_in) == 1      # and nothing of it is left behind


@pytest.mark.parametrize("name", [n for n in NAMES])
@pytest.mark.parametrize("grads", [False, True])
def test_derivatives_in_forward_mode_are_refused(stand_in, name, grads):
    fn, tensors = calls(L, "cpu")[name]
    for i, t in enumerate(tensors):
        if not t.is_floating_point():
            continue
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t.detach().clone().requires_grad_(grads), torch.ones_like(t))
            with pytest.raises(ValueError, match="forward mode"):
                fn(*tensors[:i], dual, *tensors[i + 1:])
            assert not stand_in
            fn(*tensors)      # tensors that carry none
            stand_in.clear()
