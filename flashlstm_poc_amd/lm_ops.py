"""The operators around the recurrent layers of a language model (include/flashlstm/lm_ops.h) on torch tensors: layer norm on a
residual stream, attention with a decaying state, and the distillation loss against a teacher's top logits.

Each is there as plain functions (forward, backward, and what training or serving calls in one go) and with autograd.  torch is
used for device memory, streams and autograd; every computation happens inside libflashlstm.so.  Work is enqueued on the
current stream of the tensors' device, which has to be the current device, and not waited for.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from .core import load_library

_BOUND = None
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _bind() -> ctypes.CDLL:
    """The library with the signatures of lm_ops.h."""
    global _BOUND
    if _BOUND is None:
        lib = load_library()
        vp, sz, i32, f32 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_float
        lib.flstm_layer_norm_forward.argtypes = [sz, sz, vp, sz, vp, sz, i32, vp, vp, f32, vp, vp, vp, vp, vp]
        lib.flstm_layer_norm_workspace_bytes.argtypes = [sz, sz]
        lib.flstm_layer_norm_workspace_bytes.restype = sz
        lib.flstm_layer_norm_backward.argtypes = [sz, sz, vp, sz, vp, sz, vp, sz, i32] + [vp] * 8
        _BOUND = lib
    return _BOUND


def _check(rc: int, name: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{name} failed with status {rc}")


def _device_tensor(name: str, t, dtype=None) -> int:
    """Refuses what is no tensor on the current device or of a type that the operators do not have; returns the type's code."""
    if not torch.is_tensor(t) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.get_device() != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, which is not the current device")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be of type {dtype}, not {t.dtype}")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {t.dtype} of {name}: tensors must be float32, float16 or bfloat16")
    return code


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ---- layer norm

def _rows(t):
    """`t` as (rows, width) with contiguous rows; a copy only where its layout has no such view."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check_parameter(name: str, t, width: int) -> None:
    if t is not None:
        _device_tensor(name, t, torch.float32)
        if tuple(t.shape) != (width,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of shape ({width},)")


def layer_norm_forward(x, weight=None, bias=None, *, eps: float = 1e-5, residual=None) -> Tuple:
    """total = x + residual (rounded to x's type; x itself without a residual), and the layer norm of it over the last axis.

    x, residual (..., width) float32 / float16 / bfloat16; weight, bias (width,) float32 or None.
    Returns (y, total, mean, rstd): y and total of x's shape and type, mean and rstd (rows,) float32, which
    layer_norm_backward takes."""
    code = _device_tensor("x", x)
    if x.dim() < 1:
        raise ValueError("x must have a last axis to normalise over")
    width = x.shape[-1]
    if residual is not None:
        _device_tensor("residual", residual, x.dtype)
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, not {tuple(residual.shape)}")
    _check_parameter("weight", weight, width)
    _check_parameter("bias", bias, width)
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if x.numel() == 0:
        empty = torch.empty(x.shape[:-1].numel(), device=x.device, dtype=torch.float32)
        return torch.empty_like(x), x if residual is None else torch.empty_like(x), empty, torch.empty_like(empty)
    rows_x = _rows(x)
    rows_r = None if residual is None else _rows(residual)
    rows = rows_x.shape[0]
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    total = x if residual is None else torch.empty_like(y)
    stats = torch.empty((2, rows), device=x.device, dtype=torch.float32)
    mean, rstd = stats[0], stats[1]
    _check(_bind().flstm_layer_norm_forward(rows, width, rows_x.data_ptr(), rows_x.stride(0), _ptr(rows_r),
                                            0 if rows_r is None else rows_r.stride(0), code, _ptr(weight), _ptr(bias), eps,
                                            None if residual is None else total.data_ptr(), y.data_ptr(), mean.data_ptr(),
                                            rstd.data_ptr(), _stream()), "flstm_layer_norm_forward")
    return y, total, mean, rstd


def layer_norm_backward(dy, total, weight, mean, rstd, *, d_total=None, want_parameters: bool = True) -> Tuple:
    """Gradients of layer_norm_forward from those of y and, where the stream goes on, of total (d_total).

    Returns (dx, dweight, dbias): dx (also the residual's gradient) of dy's type; dweight, dbias (width,) float32, or None
    without want_parameters."""
    code = _device_tensor("dy", dy)
    width = total.shape[-1]
    for name, t in (("total", total), ("d_total", d_total)):
        if t is not None:
            _device_tensor(name, t, dy.dtype)
            if t.shape != dy.shape:
                raise ValueError(f"{name} must have dy's shape {tuple(dy.shape)}, not {tuple(t.shape)}")
    _check_parameter("weight", weight, width)
    rows = dy.shape[:-1].numel()
    for name, t in (("mean", mean), ("rstd", rstd)):
        _device_tensor(name, t, torch.float32)
        if t.numel() != rows or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous and hold {rows} values")
    rows_dy, rows_t = _rows(dy) if dy.numel() else dy, _rows(total) if dy.numel() else total
    rows_d = None if d_total is None or not dy.numel() else _rows(d_total)
    dx = torch.empty(dy.shape, device=dy.device, dtype=dy.dtype)
    dweight = dbias = workspace = None
    lib = _bind()
    if dy.numel() == 0:
        rows = 0
    if want_parameters:
        dweight = torch.empty(width, device=dy.device, dtype=torch.float32)
        dbias = torch.empty_like(dweight)
        workspace = torch.empty(lib.flstm_layer_norm_workspace_bytes(rows, width), device=dy.device, dtype=torch.uint8)
    _check(lib.flstm_layer_norm_backward(rows, width, rows_dy.data_ptr(), rows_dy.stride(0), rows_t.data_ptr(), rows_t.stride(0),
                                         _ptr(rows_d), 0 if rows_d is None else rows_d.stride(0), code, _ptr(weight),
                                         mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), _ptr(dweight), _ptr(dbias),
                                         _ptr(workspace), _stream()), "flstm_layer_norm_backward")
    return dx, dweight, dbias


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        y, total, mean, rstd = layer_norm_forward(x, weight, bias, eps=eps, residual=residual)
        ctx.save_for_backward(total, weight, mean, rstd)
        ctx.wanted = weight is not None and ctx.needs_input_grad[2] or bias is not None and ctx.needs_input_grad[3]
        ctx.set_materialize_grads(False)
        return (y, total) if residual is not None else (y, None)

    @staticmethod
    def backward(ctx, dy, d_total):
        total, weight, mean, rstd = ctx.saved_tensors
        if dy is None:
            return d_total, d_total, None, None, None
        dx, dweight, dbias = layer_norm_backward(dy, total, weight, mean, rstd, d_total=d_total, want_parameters=ctx.wanted)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dx if need[1] else None, dweight if need[2] else None, dbias if need[3] else None, None


def layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5, residual=None):
    """layer_norm_forward with autograd: y, or with a residual (y, total)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight, bias)):
        y, total = _LayerNormFunction.apply(x, residual, weight, bias, eps)
    else:
        y, total = layer_norm_forward(x, weight, bias, eps=eps, residual=residual)[:2]
    return y if residual is None else (y, total)


class LayerNorm(torch.nn.Module):
    """Layer norm over the last axis, on a residual stream where one is handed over; parameters fp32, as torch.nn.LayerNorm
    names and initialises them.

    forward(x) -> y;  forward(x, residual) -> (y, x + residual)."""

    def __init__(self, width: int, *, eps: float = 1e-5, device="cuda"):
        super().__init__()
        if width < 1:
            raise ValueError("width must be >= 1")
        self.width, self.eps = int(width), float(eps)
        self.weight = torch.nn.Parameter(torch.ones(self.width, device=device, dtype=torch.float32))
        self.bias = torch.nn.Parameter(torch.zeros(self.width, device=device, dtype=torch.float32))

    def forward(self, x, residual=None):
        return layer_norm(x, self.weight, self.bias, eps=self.eps, residual=residual)
