"""Calls of the row-wise layers by name, as their tests make all of them."""
import torch


def calls(L, device, seed=0, rows=6):
    """{name: (function of its tensors, tensors)}; every function returns a tuple of tensors."""
    g = torch.Generator().manual_seed(seed)
    new = lambda *shape, dtype=torch.float16: torch.randn(shape, generator=g).to(device, dtype)
    codes = lambda *shape: torch.randint(-127, 128, shape, generator=g).to(device, torch.int8)
    x, w, b, r, norm = new(rows, 24), new(40, 24), new(40), new(rows, 40), new(24)
    plus = new(rows, 24)
    xs, ws = torch.rand(rows, generator=g).to(device) + 0.5, torch.rand(40, generator=g).to(device) + 0.5
    tup = lambda t: t if isinstance(t, tuple) else (t,)
    return {
        "linear": (lambda x, w, b, r: tup(L.linear(x, w, b, activation="relu", residual=r)), (x, w, b, r)),
        "linear_s8": (lambda x, xs, w, ws: tup(L.linear_s8(x, xs, w, ws, dtype=torch.float16)), (codes(rows, 24), xs, codes(40, 24), ws)),
        "rms_norm": (lambda x, w: tup(L.rms_norm(x, w)), (x, norm)),
        "rms_norm with a residual": (lambda x, w, r: tup(L.rms_norm(x, w, residual=r)), (x, norm, plus)),
        "rms_norm_s8": (lambda x, w, r: tup(L.rms_norm_s8(x, w, residual=r)), (x, norm, plus)),
        "quantize_rows": (lambda x: tup(L.quantize_rows(x)), (x,)),
    }


NAMES = ["linear", "linear_s8", "rms_norm", "rms_norm with a residual", "rms_norm_s8", "quantize_rows"]
