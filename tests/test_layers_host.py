"""What the row-wise layers refuse, and the sizes of their workspaces: nothing here is launched."""
import ctypes

import pytest
import torch

from cumm_amd import _capi
from cumm_amd import torch_layers as L

F32, S8, F16, BF16 = 0, 3, 7, 12
AT = 1 << 20      # an address that nothing reads


def linear(**more):
    a = dict(dtype=F16, out_dtype=F16, m=100, n=64, k=128, x=AT, weight=AT, out=AT, ld_x=128, ld_weight=128, ld_out=64)
    a.update(more)
    return _capi.LinearArgs(**a)


# operands that are copied: no whole pieces of 16 bytes, and products enough
COPIED = dict(m=4000, n=4096, k=4095, ld_x=4096, ld_weight=4096, ld_out=4096)


def linear_grad(**more):
    a = dict(dtype=F16, m=100, n=64, k=128, grad_out=AT, x=AT, weight=AT, ld_grad_out=64, ld_x=128, ld_weight=128, grad_x=AT, grad_weight=AT, grad_bias=AT)
    a.update(more)
    return _capi.LinearGradArgs(**a)


def norm(**more):
    a = dict(dtype=F16, m=100, k=64, x=AT, weight=AT, out=AT, ld_x=64, eps=1e-5)
    a.update(more)
    return _capi.RmsNormArgs(**a)


def norm_grad(**more):
    a = dict(dtype=F16, m=100, k=64, total=AT, weight=AT, inv_rms=AT, grad_out=AT, ld_total=64, ld_grad_out=64, grad_x=AT, grad_weight=AT)
    a.update(more)
    return _capi.RmsNormGradArgs(**a)


def refused(fn, args, text):
    with pytest.raises(ValueError, match=text):
        _capi.check(fn(ctypes.byref(args), None))


@pytest.mark.parametrize("more,text", [
    (dict(dtype=F32), "f16, bf16 or s8"), (dict(out_dtype=BF16), "the output is"), (dict(dtype=S8, out_dtype=S8), "the output is"),
    (dict(m=-1), "int32"), (dict(m=1 << 31), "int32"), (dict(n=0), "empty"), (dict(k=0), "empty"), (dict(ld_x=127), "overlap"), (dict(ld_weight=127), "overlap"),
    (dict(ld_out=63), "overlap"), (dict(residual=AT, ld_residual=63), "overlap"), (dict(pre_act=AT, ld_pre_act=63), "overlap"), (dict(ld_x=4 << 20), "8 MiB"),
    (dict(act_type=7), "activation"), (dict(act_type=-1), "activation"), (dict(x=None), "null"), (dict(weight=None), "null"), (dict(out=None), "null"),
    (dict(x=AT + 1), "aligned"), (dict(out=AT + 1), "aligned"), (dict(bias=AT + 1), "aligned"), (dict(dtype=S8), "scales"),
    (dict(dtype=S8, x_scale=AT, weight_scale=AT, k=131072, ld_x=131072, ld_weight=131072), "131071"),
    (dict(dtype=S8, x_scale=AT, weight_scale=AT, bias=AT + 2), "aligned"), (dict(m=(1 << 31) - 1, n=1 << 20, ld_out=1 << 20), "too many"),
    (dict(m=16, n=(1 << 31) - 1, ld_out=(1 << 31) - 1), "too many"),
    (dict(COPIED, workspace=AT, workspace_bytes=10), "workspace"), (COPIED, "workspace"), (dict(COPIED, workspace=AT + 16, workspace_bytes=1 << 30), "256-byte"),
])
def test_linear_refuses(more, text):
    refused(_capi.lib().cumm_hip_linear, linear(**more), text)
    if text not in ("workspace", "256-byte"):      # (what the call refuses has no size of a workspace either)
        assert _capi.lib().cumm_hip_linear_workspace(ctypes.byref(linear(**more))) == -1


@pytest.mark.parametrize("more,text", [
    (dict(dtype=S8), "f16 or bf16"), (dict(n=0), "empty"), (dict(act_type=9), "activation"), (dict(ld_grad_out=63), "overlap"), (dict(ld_x=4 << 20), "8 MiB"),
    (dict(weight=None), "needs the weight"), (dict(x=None), "needs x"), (dict(grad_out=None), "null"), (dict(act_type=4), "pre_act"),
    (dict(grad_out=AT + 1), "aligned"), (dict(), "workspace"), (dict(m=(1 << 31) - 1, k=1 << 20, ld_x=1 << 20, ld_weight=1 << 20), "too many"),
    (dict(from_inputs=1, n=60), "multiples of 8"), (dict(from_inputs=1, k=136, ld_x=136, ld_weight=136), "multiples of 8"),
    (dict(from_inputs=1, n=136, ld_grad_out=136), "multiples of 8"), (dict(from_inputs=1, act_type=5, x=None, grad_weight=None), "x and weight"),
    (dict(from_inputs=1, act_type=5, weight=None, grad_x=None), "x and weight"), (dict(from_inputs=1, bias=AT + 1), "aligned"),
    (dict(from_inputs=1, grad_x=None, x=None), "needs x"), (dict(from_inputs=1, act_type=5), "workspace"),
])
def test_linear_backward_refuses(more, text):
    refused(_capi.lib().cumm_hip_linear_backward, linear_grad(**more), text)


@pytest.mark.parametrize("more,text", [
    (dict(dtype=F32), "f16 or bf16"), (dict(dtype=S8), "f16 or bf16"), (dict(k=0), "empty"), (dict(m=-1), "empty"), (dict(ld_x=63), "overlap"),
    (dict(k=(1 << 30) + 1, ld_x=(1 << 30) + 1), "2.30"),
    (dict(eps=0.0), "eps"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(residual=AT, ld_residual=64), "sum is written"), (dict(total=AT), "sum is written"),
    (dict(x=None), "null"), (dict(out=None), "null"), (dict(codes=AT, scale=AT), "either"), (dict(out=None, codes=AT), "scale per row"), (dict(scale=AT), "scale per row"),
    (dict(weight=None), "needs its weight"), (dict(weight=None, codes=AT, out=None, scale=AT, inv_rms=AT), "without a norm"), (dict(x=AT + 1), "aligned"),
    (dict(dtype=F32, weight=None, out=None, codes=AT, scale=AT, x=AT + 2), "aligned"),
])
def test_norm_refuses(more, text):
    refused(_capi.lib().cumm_hip_rms_norm, norm(**more), text)


@pytest.mark.parametrize("more,text", [
    (dict(dtype=F32), "f16 or bf16"), (dict(k=0), "empty"), (dict(ld_total=63), "overlap"), (dict(total=None), "null"), (dict(inv_rms=None), "null"),
    (dict(grad_x=AT + 1), "aligned"), (dict(), "workspace"),
])
def test_norm_backward_refuses(more, text):
    refused(_capi.lib().cumm_hip_rms_norm_backward, norm_grad(**more), text)


def test_null_arguments():
    lib = _capi.lib()
    for name in ("linear", "linear_backward", "rms_norm", "rms_norm_backward"):
        assert getattr(lib, "cumm_hip_" + name)(None, None) == _capi.EINVAL
    for name in ("linear", "linear_backward", "rms_norm_backward"):
        assert getattr(lib, "cumm_hip_%s_workspace" % name)(None) == -1


def test_no_rows_are_no_work():
    lib = _capi.lib()
    assert lib.cumm_hip_linear(ctypes.byref(linear(m=0, x=None, out=None)), None) == 0
    assert lib.cumm_hip_rms_norm(ctypes.byref(norm(m=0, x=None)), None) == 0
    assert lib.cumm_hip_linear_workspace(ctypes.byref(linear(m=0))) == 0
    assert lib.cumm_hip_linear_backward_workspace(ctypes.byref(linear_grad(m=0))) == 0


def test_workspaces():
    """Operands that lie on 16-byte borders and are whole pieces long are read in place; others too, or copied to lines of 128
    bytes, whichever takes less time; the gradient through an activation is kept for the two products."""
    lib = _capi.lib()
    need = lambda **m: lib.cumm_hip_linear_workspace(ctypes.byref(linear(**m)))
    assert need(m=16) == 0
    assert need(m=16, k=127) == need(m=16, x=AT + 2) == need(m=16, ld_weight=129) == 0
    assert need(m=16, k=7) == 16 * 128 + 64 * 128               # (less than a piece)
    assert need(**COPIED) == 4000 * 8192 + 4096 * 8192          # both: 4095 elements are no whole pieces
    assert need(**dict(COPIED, k=4096, x=AT + 2)) == 4000 * 8192      # x alone
    assert need(**dict(COPIED, k=4096, ld_weight=4097)) == 4096 * 8192
    back = lambda **m: lib.cumm_hip_linear_backward_workspace(ctypes.byref(linear_grad(**dict(dict(grad_weight=None, grad_bias=None), **m))))
    plain = back()
    assert back(act_type=4, pre_act=AT, ld_pre_act=64) == plain + 100 * 64 * 2      # (100 rows of 64: 12800 bytes, 50 times 256)
    narrow = back(from_inputs=1, act_type=4)
    assert narrow == 64 * (128 + 1) * 4                         # one workgroup's sums: 100 rows are fewer than 128
    assert back(from_inputs=1, act_type=4, m=129) == 2 * narrow and back(from_inputs=1, act_type=4, m=1 << 30) == 256 * narrow
    assert lib.cumm_hip_rms_norm_backward_workspace(ctypes.byref(norm_grad())) % (64 * 4) == 0
    assert lib.cumm_hip_rms_norm_backward_workspace(ctypes.byref(norm_grad(grad_weight=None))) == 0


def test_struct_sizes_match_the_header(tmp_path):
    import os
    import shutil
    import subprocess
    sizes = [ctypes.sizeof(c) for c in (_capi.LinearArgs, _capi.LinearGradArgs, _capi.RmsNormArgs, _capi.RmsNormGradArgs)]
    if shutil.which("gcc"):
        src = tmp_path / "sz.c"
        src.write_text('#include <stdio.h>\n#include "cumm_hip.h"\nint main(){printf("%zu %zu %zu %zu", sizeof(CummHipLinearArgs), '
                       "sizeof(CummHipLinearGradArgs), sizeof(CummHipRmsNormArgs), sizeof(CummHipRmsNormGradArgs));}\n")
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        exe = str(tmp_path / "sz")
        subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", exe])
        assert [int(x) for x in subprocess.check_output([exe]).split()] == sizes


def test_tensors_are_checked():
    h = torch.zeros(4, 8, dtype=torch.float16)
    w = torch.zeros(6, 8, dtype=torch.float16)
    q, s = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    for call, text in [
            (lambda: L.linear(h, w), "on the GPU"), (lambda: L.linear(h.float(), w.float()), "float16 or bfloat16"), (lambda: L.linear(h, w.bfloat16()), "same dtype"),
            (lambda: L.linear(h, w[:, :7]), r"weight \[N, K\]"), (lambda: L.linear(h, w[:0]), r"weight \[N, K\]"), (lambda: L.linear(h[:, :0], w[:, :0]), r"weight \[N, K\]"),
            (lambda: L.linear_s8(h, s, q, s), "int8"), (lambda: L.linear_s8(q, s, q, s, dtype=torch.float32), "dtype must be"),
            (lambda: L.linear_s8(q, s[:3], q, s), "x_scale"), (lambda: L.linear_s8(q, s, q, s.double()), "weight_scale"), (lambda: L.linear_s8(q, s, q, s), "on the GPU"),
            (lambda: L.rms_norm(h, h[0]), "on the GPU"), (lambda: L.rms_norm(h.float(), h[0].float()), "float16 or bfloat16"), (lambda: L.rms_norm(h, h[0, :7]), "weight must be"),
            (lambda: L.rms_norm(h, h[0], 0.0), "eps"), (lambda: L.rms_norm(h, h[0].bfloat16()), "weight must be"), (lambda: L.quantize_rows(q), "must be float16"),
            (lambda: L.quantize_rows(h), "on the GPU"), (lambda: L.quantize_rows(h.float().requires_grad_()), "no gradient"),
            (lambda: L.rms_norm_s8(h, h[0].clone().requires_grad_()), "no gradient")]:
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(ValueError, match="activation"):
        L.Linear(8, 8, activation="tanh", device="cpu")
