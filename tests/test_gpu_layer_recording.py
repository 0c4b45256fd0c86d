"""Calls of the row-wise layers that somebody records, on the GPU: see test_layers_recording."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from layers_calls import NAMES, calls

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


@pytest.mark.parametrize("name,grads", [(n, False) for n in NAMES] + [(n, True) for n in NAMES if "s8" not in n and n != "quantize_rows"])
def test_traces_compute(L, name, grads):
    fn, tensors = calls(L, "cuda")[name]
    leaf = lambda tensors: tuple(t.requires_grad_(grads) if t.is_floating_point() else t for t in tensors)
    with torch.set_grad_enabled(grads):
        traced = torch.jit.trace(fn, leaf(tensors), check_trace=False)
        for seed in (1, 2):
            more = leaf(calls(L, "cuda", seed=seed, rows=9)[name][1])
            assert all(torch.equal(a, b) for a, b in zip(traced(*more), fn(*more)))


@pytest.mark.parametrize("name", NAMES)
def test_what_would_leave_the_launch_out_is_refused(L, name):
    from torch.fx.experimental.proxy_tensor import make_fx
    fn, tensors = calls(L, "cuda")[name]
    want = fn(*tensors)
    with pytest.raises(ValueError, match="recorded"):
        make_fx(fn)(*tensors)
    for i, t in enumerate(tensors):
        if t.is_floating_point():
            with forward_ad.dual_level():
                with pytest.raises(ValueError, match="forward mode"):
                    fn(*tensors[:i], forward_ad.make_dual(t, torch.ones_like(t)), *tensors[i + 1:])
    assert all(torch.equal(a, b) for a, b in zip(fn(*tensors), want))
