"""Gates of the row-wise layers whose activation has a kink: what is refused, and the sizes of workspaces.  Nothing here is launched."""
import ctypes

import pytest

from cumm_amd import _capi
from test_layers_host import AT, BF16, F16, S8, linear, linear_grad, refused

NARROW = dict(k=64, ld_x=64, ld_weight=64)


@pytest.mark.parametrize("more", [dict(act_type=0), dict(act_type=4), dict(act_type=1, n=136, ld_out=136), dict(act_type=1, n=60), dict(act_type=3, k=136, ld_x=136, ld_weight=136),
                                  dict(act_type=1, dtype=S8, x_scale=AT, weight_scale=AT)])
def test_gates_are_of_few_channels_with_a_kink(more):
    refused(_capi.lib().cumm_hip_linear, linear(**dict(NARROW, gate=AT, **more) if "k" not in more else dict(more, gate=AT)), "gate")


def test_gates_are_refused_elsewhere():
    lib = _capi.lib()
    refused(lib.cumm_hip_linear, linear(gate=AT + 2, act_type=1, **NARROW), "aligned")
    refused(lib.cumm_hip_linear_backward, linear_grad(gate=AT, act_type=1, pre_act=AT, ld_pre_act=64, **NARROW), "from_inputs")
    refused(lib.cumm_hip_linear_backward, linear_grad(gate=AT, act_type=4, from_inputs=1, **NARROW), "a gate is that of")
    refused(lib.cumm_hip_linear_backward, linear_grad(gate=AT + 1, act_type=1, from_inputs=1, **NARROW), "aligned")
    refused(lib.cumm_hip_linear_backward, linear_grad(gate=AT, act_type=1, from_inputs=1, x=None, **NARROW), "needs x")
    refused(lib.cumm_hip_linear_backward, linear_grad(act_type=1, from_inputs=1, weight=None, grad_x=None, **NARROW), "x and weight")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_workspaces(dtype):
    lib = _capi.lib()
    assert lib.cumm_hip_linear_workspace(ctypes.byref(linear(dtype=dtype, out_dtype=dtype, m=5000, act_type=1, ld_x=129, x=AT + 2))) == 0
    size = lambda **more: lib.cumm_hip_linear_backward_workspace(ctypes.byref(linear_grad(dtype=dtype, from_inputs=1, **more)))
    kept, made = size(act_type=1, gate=AT), size(act_type=1)
    assert kept == size(act_type=4) and made == kept + 1024      # (100 rows of 8 bytes, up to 256)
    assert size(act_type=3, gate=AT, x=None, weight=None, grad_x=None, grad_weight=None) == kept
