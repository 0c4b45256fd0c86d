"""Sizes at the limits of a launch: a product is refused only where no kernel can run it.  Nothing here is launched."""
import ctypes

import pytest

from cumm_amd import _capi
from test_layers_host import AT, BF16, F16, S8, linear, linear_grad, refused

MOST = 256 * ((1 << 23) - 1)      # rows, or columns, of 2^23 - 1 tiles


def workspace(**more):
    return _capi.lib().cumm_hip_linear_workspace(ctypes.byref(linear(**more)))


@pytest.mark.parametrize("m,n", [(1, 1 << 27), (16, 1 << 27), (17, 1 << 27), (33, 1 << 28), (1, 1 << 30), (16, MOST), (64, MOST), (65, MOST), (MOST, 1), (1 << 30, 8),
                                 (MOST, 256), (1 << 30, 250), (1 << 20, 1 << 17)])
@pytest.mark.parametrize("dtype", [F16, BF16, S8])
def test_sizes_that_some_kernel_runs(dtype, m, n):
    k = 16
    more = dict(dtype=dtype, out_dtype=F16 if dtype == S8 else dtype, m=m, n=n, k=k, ld_x=k, ld_weight=k, ld_out=n)
    if dtype == S8:
        more.update(x_scale=AT, weight_scale=AT)
    assert workspace(**more) >= 0
    for lead in (2, 8):      # rows that have to be copied, or read as they lie
        assert workspace(**dict(more, x=AT + lead, ld_x=k + 1)) >= 0


@pytest.mark.parametrize("m,n", [((1 << 31) - 1, 1), (MOST + 1, 1), (1, (1 << 31) - 1), (257, 1 << 30), (1 << 30, 1 << 10), (MOST, 257)])
def test_sizes_that_none_runs(m, n):
    refused(_capi.lib().cumm_hip_linear, linear(m=m, n=n, k=16, ld_x=16, ld_weight=16, ld_out=n), "too many")
    assert workspace(m=m, n=n, k=16, ld_x=16, ld_weight=16, ld_out=n) == -1


@pytest.mark.parametrize("m,n,k", [(1 << 30, 136, 8), (1 << 30, 8, 136), (MOST, 136, 8), (MOST, 8, 256)])
def test_backward_passes_that_some_kernel_runs(m, n, k):
    more = dict(m=m, n=n, k=k, ld_grad_out=n, ld_x=k, ld_weight=k)
    assert _capi.lib().cumm_hip_linear_backward_workspace(ctypes.byref(linear_grad(**more))) >= 0
    refused(_capi.lib().cumm_hip_linear_backward, linear_grad(**dict(more, m=(1 << 31) - 1)), "too many")


@pytest.mark.parametrize("act", [1, 3])
def test_few_channels_with_a_kink_have_no_such_limit(act):
    assert workspace(m=(1 << 31) - 1, n=128, k=128, act_type=act, ld_out=128) == 0
