"""Row-wise layers for torch tensors, beside the sparse convolutions of ``torch_bridge``: a matrix product with bias,
activation and residual in its epilogue, the root-mean-square norm with the residual's addition, rows in 8 bits with a scale
each, and the product of such rows.  Every computing kernel, of the gradients too, is this library's (``cumm_hip_linear``,
``cumm_hip_rms_norm`` and their backward passes in ``include/cumm_hip.h``).  The reference has no layer of this kind.

Tensors are f16 or bf16 on one GPU, of any number of leading dimensions; the last one is the row.  Rows may be any number of
elements apart; a tensor whose rows are not contiguous, or whose leading dimensions are not one run of rows, is copied.
Calls go to the current stream of the tensors' device and allocate from torch's caching allocator: they can be captured
into graphs.  ``torch.jit.trace`` records a call as a Python operator; forward-mode derivatives and make_fx, which would see the
allocations and not the launch, are refused.  A failed check raises ValueError, a failed launch RuntimeError.
"""
import ctypes
import sys
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _capi, torch_bridge
from . import tensorview as tv

ACTIVATIONS = {"none": 0, "relu": 1, "sigmoid": 2, "leaky_relu": 3, "silu": 4, "gelu": 5, "gelu_tanh": 6}
_TYPES = {torch.float16: int(tv.float16), torch.bfloat16: int(tv.bfloat16), torch.int8: int(tv.int8), torch.float32: int(tv.float32)}
_KINKS = (ACTIVATIONS["relu"], ACTIVATIONS["leaky_relu"])
_HALVES = (torch.float16, torch.bfloat16)


def _check(ok: bool, text: str) -> None:
    if not ok:
        raise ValueError(text)


def _native():
    """The native half (csrc/torch_layers.h), which makes the calls that it can: everything else, and all of them where there
    is none, is made here."""
    if torch._C._are_functorch_transforms_active() or torch.compiler.is_compiling():
        return None
    return torch_bridge._native()


def _not_recorded(name: str, *tensors) -> None:
    """Refuses what would leave the launch out and say nothing: a derivative in forward mode, a graph of torch's operators."""
    if torch.autograd.forward_ad._current_level >= 0 and any(
            t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("%s has no derivative in forward mode" % name)
    proxies = sys.modules.get("torch.fx.experimental.proxy_tensor")
    if proxies is not None and proxies.get_proxy_mode() is not None:
        raise ValueError("%s cannot be recorded as torch operators" % name)


def _differentiable(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _Recorded(torch.autograd.Function):
    """A call without a gradient where ``torch.jit.trace`` records: a Python operator in its graph."""

    @staticmethod
    def forward(ctx, fn, *args):
        out = fn(*args)
        ctx.mark_non_differentiable(*(out if isinstance(out, tuple) else (out,)))
        return out


def _made(fn, *args):
    return _Recorded.apply(fn, *args) if torch.jit.is_tracing() else fn(*args)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as a matrix of its rows, without a copy where the rows are contiguous and evenly apart, by less than the 8 MiB that
    a product takes."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] > 1 or t.shape[0] > 1 and not t.shape[1] <= t.stride(0) < (8 << 20) // t.element_size():
        t = t.contiguous()
    return t


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _on_device(first: torch.Tensor, **others) -> None:
    _check(first.is_cuda, "tensors must be on the GPU")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError("%s is on %s, not on %s" % (name, t.device, first.device))


def _kept(name: str, t: torch.Tensor, like: torch.Tensor, dtype, *shape) -> torch.Tensor:
    """A tensor that was kept for the backward pass, as it comes back: an unpack hook may give another one."""
    _check(t.device == like.device and t.dtype == dtype and t.shape == shape,
           "the tensor kept as %s came back as %s %s on %s, not as %s %s on %s" % (name, t.dtype, tuple(t.shape), t.device, dtype, shape, like.device))
    return t


class _Device:
    """The device of a call's tensors, where it is not the current one."""

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.back = torch.cuda.current_device()
        if self.back != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *_):
        if self.back != self.index:
            torch.cuda.set_device(self.back)


def _stream() -> int:
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _call(fn, query, args, device) -> None:
    """The call with a workspace of the size that it asks for."""
    need = query(ctypes.byref(args)) if query is not None else 0
    ws = None
    if need > 0:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
    status = fn(ctypes.byref(args), _stream())
    if status:
        _capi.check(status)


# ---- linear

def _linear_forward(x, weight, bias, residual, act, slope, scales, dtype, want_pre, gate=None):
    """(out, pre_act or None) for matrices."""
    lib = _capi.lib()
    m, k, n = x.shape[0], x.shape[1], weight.shape[0]
    with _Device(x.device):
        out = torch.empty((m, n), dtype=dtype, device=x.device)
        pre = torch.empty_like(out) if want_pre else None
        a = _capi.LinearArgs()
        a.dtype, a.out_dtype, a.m, a.n, a.k = _TYPES[x.dtype], _TYPES[dtype], m, n, k
        a.x, a.weight, a.bias, a.residual = x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(residual)
        a.out, a.pre_act, a.gate = out.data_ptr(), _ptr(pre), _ptr(gate)
        a.ld_x, a.ld_weight, a.ld_out, a.ld_pre_act = _pitch(x), _pitch(weight), n, n
        if residual is not None:
            a.ld_residual = _pitch(residual)
        if scales is not None:
            a.x_scale, a.weight_scale = scales[0].data_ptr(), scales[1].data_ptr()
        a.act_type, a.act_alpha = act, slope
        _call(lib.cumm_hip_linear, lib.cumm_hip_linear_workspace, a, x.device)
    return out, pre


def _linear_result(x, weight, bias, residual, act, slope, x_scale, weight_scale, dtype):
    return _linear_forward(x, weight, bias, residual, act, slope, None if x_scale is None else (x_scale, weight_scale), dtype, False)[0]


class _Linear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act: int, slope: float):
        # what the backward pass needs of the activation's argument.  Of few channels it is worked out again, or, where only its side
        # of a kink counts, kept as a bit; the sign of a ReLU's result is that of its argument, unless something is added to it
        ctx.again = all(c % 8 == 0 and c <= _capi.LINEAR_NARROW for c in weight.shape)
        ctx.kink = ctx.again and act in _KINKS
        whole = ctx.again and act != 0 and not ctx.kink
        by_result = act == ACTIVATIONS["relu"] and residual is None and not ctx.again
        gate = None
        if ctx.kink:
            gate = torch.empty(x.shape[0], _capi.LINEAR_GATE_BYTES(weight.shape[0]), dtype=torch.uint8, device=x.device)
        out, pre = _linear_forward(x, weight, bias, residual, act, slope, None, x.dtype, act != 0 and not by_result and not ctx.again, gate)
        ctx.act, ctx.slope, ctx.k = act, slope, weight.shape[1]
        ctx.save_for_backward(x if ctx.needs_input_grad[1] or whole else None, weight if ctx.needs_input_grad[0] or whole else None,
                              gate if ctx.kink else (bias if whole else (out if by_result else pre)))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, pre = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        grad_x = grad_w = grad_b = None
        if need_x or need_w or need_b:
            lib, g = _capi.lib(), _rows(grad)
            m, n = g.shape
            k = ctx.k
            with _Device(g.device):
                a = _capi.LinearGradArgs()
                a.dtype, a.m, a.n, a.k, a.grad_out, a.ld_grad_out = _TYPES[g.dtype], m, n, k, g.data_ptr(), _pitch(g)
                a.from_inputs = ctx.again
                if ctx.kink:
                    pre = _kept("gate", pre, g, torch.uint8, m, _capi.LINEAR_GATE_BYTES(n)).contiguous()
                    a.gate = pre.data_ptr()
                elif pre is not None and ctx.again:
                    pre = _kept("bias", pre, g, g.dtype, n).contiguous()
                    a.bias = pre.data_ptr()
                elif pre is not None:
                    pre = _rows(_kept("the activation's argument", pre, g, g.dtype, m, n))
                    a.pre_act, a.ld_pre_act = pre.data_ptr(), _pitch(pre)
                a.act_type, a.act_alpha = ctx.act, ctx.slope
                if x is not None:
                    x = _rows(_kept("x", x, g, g.dtype, m, k))
                    a.x, a.ld_x = x.data_ptr(), _pitch(x)
                if weight is not None:
                    weight = _rows(_kept("weight", weight, g, g.dtype, n, k))
                    a.weight, a.ld_weight = weight.data_ptr(), _pitch(weight)
                if need_x:
                    grad_x = torch.empty((m, k), dtype=g.dtype, device=g.device)
                    a.grad_x = grad_x.data_ptr()
                if need_w:
                    grad_w = torch.empty((n, k), dtype=g.dtype, device=g.device)
                    a.grad_weight = grad_w.data_ptr()
                if need_b:
                    grad_b = torch.empty(n, dtype=g.dtype, device=g.device)
                    a.grad_bias = grad_b.data_ptr()
                _call(lib.cumm_hip_linear_backward, lib.cumm_hip_linear_backward_workspace, a, g.device)
        return grad_x, grad_w, grad_b, grad if need_r else None, None, None


def _linear_args(name, x, weight, bias, residual, activation, out_dtype, bias_dtype):
    _check(x.dim() >= 1 and weight.dim() == 2 and weight.shape[1] == x.shape[-1] and weight.shape[0] > 0 and weight.shape[1] > 0,
           "%s: x must be [..., K] and weight [N, K]" % name)
    _check(max(weight.shape) < 1 << 31, "%s: sizes must not exceed int32 range" % name)
    _check(weight.dtype == x.dtype, "%s: x and weight must have the same dtype" % name)
    _on_device(x, weight=weight, bias=bias, residual=residual)
    n = weight.shape[0]
    if bias is not None:
        _check(bias.shape == (n,) and bias.dtype == bias_dtype, "%s: bias must be [%d] of %s" % (name, n, bias_dtype))
        bias = bias.contiguous()
    if residual is not None:
        _check(residual.shape == x.shape[:-1] + (n,) and residual.dtype == out_dtype,
               "%s: residual must have the shape of the result and be %s" % (name, out_dtype))
        residual = _rows(residual)
    act = ACTIVATIONS.get(activation)
    _check(act is not None, "%s: activation must be one of %s" % (name, ", ".join(ACTIVATIONS)))
    return _rows(x), _rows(weight), bias, residual, act


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: str = "none",
           residual: Optional[torch.Tensor] = None, slope: float = 0.01) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` for x [..., K], weight [N, K] (f16 / bf16); the result is rounded
    once.  Differentiable in all four tensors (once): the gradient of what the activation got is rounded to the tensors' type
    before its products with weight and x, and so is what the activation got where it is kept.  With N and K multiples of 8 up to
    128 it is worked out again from x, weight and bias, which are kept for that, or, for "relu" and "leaky_relu", which elements pass is
    kept, a bit each, decided by the exact sign of the activation's argument.  ``slope`` is that of "leaky_relu"."""
    native = _native()
    if native is not None and activation in ACTIVATIONS:
        out = native.layer_linear(x, weight, bias, residual, ACTIVATIONS[activation], slope)
        if out is not None:
            return out
    _not_recorded("linear", x, weight, bias, residual)
    _check(x.dtype in _HALVES, "linear: x must be float16 or bfloat16 (linear_s8 takes 8-bit rows)")
    shape = x.shape[:-1] + weight.shape[:1]
    x, weight, bias, residual, act = _linear_args("linear", x, weight, bias, residual, activation, x.dtype, x.dtype)
    if _differentiable(x, weight, bias, residual):
        out = _Linear.apply(x, weight, bias, residual, act, slope)
    else:
        out = _made(_linear_result, x, weight, bias, residual, act, slope, None, None, x.dtype)
    return out if out.shape == shape else out.view(shape)


def linear_s8(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
              bias: Optional[torch.Tensor] = None, *, activation: str = "none", residual: Optional[torch.Tensor] = None,
              slope: float = 0.01, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The same for 8-bit rows: x [..., K] and weight [N, K] int8 with the scales of their rows (float32: x_scale [...],
    weight_scale [N], as ``quantize_rows`` and ``rms_norm_s8`` give them), bias float32, residual and result ``dtype``.
    Inference only: it has no gradient.  K up to 131071 (the sums of products are whole numbers of 32 bits)."""
    native = _native()
    if native is not None and activation in ACTIVATIONS:
        out = native.layer_linear_s8(x, x_scale, weight, weight_scale, bias, residual, ACTIVATIONS[activation], slope, dtype)
        if out is not None:
            return out
    _check(x.dtype == torch.int8, "linear_s8: x must be int8")
    _check(dtype in _HALVES, "linear_s8: dtype must be float16 or bfloat16")
    shape = x.shape[:-1] + weight.shape[:1]
    _check(x_scale.dtype == torch.float32 and x_scale.shape == x.shape[:-1], "linear_s8: x_scale must be float32, one per row of x")
    _check(weight_scale.dtype == torch.float32 and weight_scale.shape == weight.shape[:1],
           "linear_s8: weight_scale must be float32, one per row of weight")
    _on_device(x, x_scale=x_scale, weight_scale=weight_scale)
    _no_gradient("linear_s8", x_scale, weight_scale, bias, residual)
    x, weight, bias, residual, act = _linear_args("linear_s8", x, weight, bias, residual, activation, dtype, torch.float32)
    return _made(_linear_result, x, weight, bias, residual, act, slope, x_scale.contiguous(), weight_scale.contiguous(), dtype).view(shape)


# ---- norms

def _norm_forward(x, weight, residual, eps, codes: bool, want_inv: bool):
    """(out or codes, scale, total, inv) for matrices; None where there is none."""
    lib = _capi.lib()
    m, k = x.shape
    with _Device(x.device):
        new = lambda dtype, *shape: torch.empty(shape, dtype=dtype, device=x.device)
        out = new(torch.int8 if codes else x.dtype, m, k)
        scale = new(torch.float32, m) if codes else None
        total = new(x.dtype, m, k) if residual is not None else None
        inv = new(torch.float32, m) if want_inv else None
        a = _capi.RmsNormArgs()
        a.dtype, a.m, a.k, a.eps = _TYPES[x.dtype], m, k, eps
        a.x, a.ld_x, a.weight = x.data_ptr(), _pitch(x), _ptr(weight)
        if residual is not None:
            a.residual, a.ld_residual, a.total = residual.data_ptr(), _pitch(residual), total.data_ptr()
        if codes:
            a.codes, a.scale = out.data_ptr(), scale.data_ptr()
        else:
            a.out = out.data_ptr()
        a.inv_rms = _ptr(inv)
        _call(lib.cumm_hip_rms_norm, None, a, x.device)
    return out, scale, total, inv


def _norm_result(x, weight, residual, eps, codes):
    """What the caller gets: out or codes, then scale and total where there are."""
    got = tuple(t for t in _norm_forward(x, weight, residual, eps, codes, False)[:3] if t is not None)
    return got if len(got) > 1 else got[0]


class _RmsNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, residual, eps: float):
        out, _, total, inv = _norm_forward(x, weight, residual, eps, False, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if total is None else total, weight, inv)
        return out if total is None else (out, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_total=None):
        total, weight, inv = ctx.saved_tensors
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if grad is None and grad_total is None:
            return None, None, None, None
        like = grad if grad is not None else grad_total      # (of the result's shape and type, as x)
        m, k = like.shape
        total = _rows(_kept("the normed rows", total, like, like.dtype, m, k))
        weight = _kept("weight", weight, like, like.dtype, k).contiguous()
        inv = _kept("the rows' statistics", inv, like, torch.float32, m).contiguous()
        lib = _capi.lib()
        grad_x = grad_w = None
        with _Device(total.device):
            a = _capi.RmsNormGradArgs()
            a.dtype, a.m, a.k = _TYPES[total.dtype], m, k
            a.total, a.ld_total, a.weight, a.inv_rms = total.data_ptr(), _pitch(total), weight.data_ptr(), inv.data_ptr()
            if grad is not None:
                grad = _rows(grad)
                a.grad_out, a.ld_grad_out = grad.data_ptr(), _pitch(grad)
            if grad_total is not None:
                grad_total = _rows(grad_total)
                a.grad_total, a.ld_grad_total = grad_total.data_ptr(), _pitch(grad_total)
            if need_x or need_r:
                grad_x = torch.empty((m, k), dtype=total.dtype, device=total.device)
                a.grad_x = grad_x.data_ptr()
            if need_w:
                grad_w = torch.empty(k, dtype=total.dtype, device=total.device)
                a.grad_weight = grad_w.data_ptr()
            _call(lib.cumm_hip_rms_norm_backward, lib.cumm_hip_rms_norm_backward_workspace, a, total.device)
        return grad_x if need_x else None, grad_w, grad_x if need_r else None, None


def _norm_args(name, x, weight, residual, eps):
    _check(x.dim() >= 1 and 0 < x.shape[-1] < 1 << 31, "%s: x must be [..., K]" % name)
    _check(x.dtype in _HALVES, "%s: x must be float16 or bfloat16" % name)
    _check(weight.shape == x.shape[-1:] and weight.dtype == x.dtype, "%s: weight must be [%d] of %s" % (name, x.shape[-1], x.dtype))
    _check(eps > 0, "%s: eps must be positive" % name)
    _on_device(x, weight=weight, residual=residual)
    if residual is not None:
        _check(residual.shape == x.shape and residual.dtype == x.dtype, "%s: residual must have the shape and dtype of x" % name)
        residual = _rows(residual)
    return _rows(x), weight.contiguous(), residual


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
             residual: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``h / sqrt(mean(h^2) + eps) * weight`` over the last dimension of ``h = x``; with a residual ``h = x + residual``, rounded
    to the tensors' type, and (result, h) comes back.  Differentiable in all tensors (once)."""
    native = _native()
    if native is not None:
        got = native.layer_norm(x, weight, residual, eps, False)
        if got is not None:
            return got
    _not_recorded("rms_norm", x, weight, residual)
    shape = x.shape
    x, weight, residual = _norm_args("rms_norm", x, weight, residual, eps)
    if _differentiable(x, weight, residual):
        got = _RmsNorm.apply(x, weight, residual, eps)
    else:
        got = _made(_norm_result, x, weight, residual, eps, False)
    if residual is None:
        return got.view(shape)
    return got[0].view(shape), got[1].view(shape)


def rms_norm_s8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, residual: Optional[torch.Tensor] = None):
    """The norm with its result in 8 bits: (codes int8, scale float32 of every row), and h with a residual; code * scale
    stands for the result.  A row's largest magnitude is 127; a row of zeros has scale 0, one with an infinity or a NaN a scale
    that is not finite.  Inference only."""
    native = _native()
    if native is not None:
        got = native.layer_norm(x, weight, residual, eps, True)
        if got is not None:
            return got
    _no_gradient("rms_norm_s8", x, weight, residual)
    shape = x.shape
    x, weight, residual = _norm_args("rms_norm_s8", x, weight, residual, eps)
    codes, scale, *total = _made(_norm_result, x, weight, residual, eps, True)
    return (codes.view(shape), scale.view(shape[:-1])) + tuple(t.view(shape) for t in total)


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] (f16, bf16 or f32) in 8 bits: (codes int8, scale float32 [...]), as ``rms_norm_s8`` gives them.  For weights
    [N, K] of ``linear_s8`` and activations between two products."""
    native = _native()
    if native is not None:
        got = native.layer_quantize(x)
        if got is not None:
            return got
    _no_gradient("quantize_rows", x)
    _check(x.dim() >= 1 and 0 < x.shape[-1] < 1 << 31, "quantize_rows: x must be [..., K]")
    _check(x.dtype in _HALVES or x.dtype == torch.float32, "quantize_rows: x must be float16, bfloat16 or float32")
    _on_device(x)
    shape = x.shape
    codes, scale = _made(_norm_result, _rows(x), None, None, 1.0, True)
    return codes.view(shape), scale.view(shape[:-1])


def _no_gradient(name, *tensors):
    _not_recorded(name, *tensors)
    if _differentiable(*tensors):
        raise ValueError("%s has no gradient: call it under torch.no_grad()" % name)


class Linear(torch.nn.Module):
    """A layer over :func:`linear`."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str = "none", slope: float = 0.01,
                 dtype=torch.float16, device="cuda"):
        super().__init__()
        _check(activation in ACTIVATIONS, "activation must be one of %s" % ", ".join(ACTIVATIONS))
        w = torch.randn(out_features, in_features, device=device) / in_features ** 0.5
        self.weight = torch.nn.Parameter(w.to(dtype))
        self.bias = torch.nn.Parameter(torch.zeros(out_features, dtype=dtype, device=device)) if bias else None
        self.activation, self.slope = activation, slope

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return linear(x, self.weight, self.bias, activation=self.activation, residual=residual, slope=self.slope)


class RMSNorm(torch.nn.Module):
    """A layer over :func:`rms_norm`."""

    def __init__(self, features: int, eps: float = 1e-6, dtype=torch.float16, device="cuda"):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(features, dtype=dtype, device=device))
        self.eps = eps

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(x, self.weight, self.eps, residual=residual)
