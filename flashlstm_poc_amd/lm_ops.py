"""The operators around the recurrent layers of a language model (include/flashlstm/lm_ops.h) on torch tensors: layer norm on a
residual stream, attention with a decaying state, the distillation loss against a teacher's top logits, the embedding of tokens, a gated
linear recurrence, and beam search.

Each but the last is there as plain functions (forward, backward, and what training or serving calls in one go) and with autograd, which has
no forward-mode derivatives of them and says so.  torch is used for device memory, streams and autograd; every computation happens
inside libflashlstm.so.  Work is enqueued on the current stream of the tensors' device, which has to be the current device, and
not waited for.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

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
        rows = shape = ctypes.c_char_p   # (packed structures)
        lib.flstm_decay_attention_forward.argtypes = [shape, rows, rows, rows, vp, rows, vp, vp, vp]
        lib.flstm_decay_attention_backward.argtypes = [shape, rows, rows, rows, rows, vp, vp, rows, rows, rows, vp, vp, vp]
        lib.flstm_decay_attention_workspace_bytes.argtypes = [shape, i32]
        lib.flstm_decay_attention_workspace_bytes.restype = sz
        lib.flstm_decay_attention_step.argtypes = [shape, rows, rows, rows, rows, vp, vp]
        problem = ctypes.c_char_p
        lib.flstm_distillation_forward.argtypes = [problem, vp, vp, vp]
        lib.flstm_distillation_backward.argtypes = [problem, vp, vp, sz, vp, sz, vp]
        lib.flstm_distillation_workspace_bytes.argtypes = [problem]
        lib.flstm_distillation_workspace_bytes.restype = sz
        lib.flstm_distillation_train.argtypes = [problem, vp, sz, vp, vp, sz, vp, vp]
        lib.flstm_embedding_forward.argtypes = [problem, vp, sz, i32, vp, i32, vp]
        lib.flstm_embedding_workspace_bytes.argtypes = [problem]
        lib.flstm_embedding_workspace_bytes.restype = sz
        lib.flstm_embedding_backward.argtypes = [problem, vp, sz, i32, vp, i32, vp, vp]
        lib.flstm_gated_recurrence_forward.argtypes = [shape, rows, rows, rows, vp, rows, vp, vp, vp, vp]
        lib.flstm_gated_recurrence_backward.argtypes = [shape, rows, rows, rows, rows, vp, vp, rows, rows, rows, vp, vp, vp]
        lib.flstm_gated_recurrence_step.argtypes = [shape, rows, rows, rows, rows, vp, vp]
        lib.flstm_gated_recurrence_workspace_bytes.argtypes = [shape, i32]
        lib.flstm_gated_recurrence_workspace_bytes.restype = sz
        lib.flstm_gated_recurrence_saved_rows.argtypes = [shape]
        lib.flstm_gated_recurrence_saved_rows.restype = sz
        lib.flstm_beam_select.argtypes = [problem, vp, vp, vp, vp, vp, vp]
        lib.flstm_beam_select_workspace_bytes.argtypes = [problem]
        lib.flstm_beam_select_workspace_bytes.restype = sz
        lib.flstm_beam_reorder.argtypes = [sz, i32, vp, ctypes.c_char_p, i32, vp]
        _BOUND = lib
    return _BOUND


def _check(rc: int, name: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{name} failed with status {rc}")


def _device_tensor(name: str, t, dtype=None) -> int:
    """Refuses what is no tensor on the current device or of a type that the operators do not have; returns the type's code."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"{name} is on {t.device}, which is not the current device")
    kind = t.dtype
    if dtype is not None and kind != dtype:
        raise ValueError(f"{name} must be of type {dtype}, not {kind}")
    code = _DTYPES.get(kind)
    if code is None:
        raise ValueError(f"unsupported dtype {kind} of {name}: tensors must be float32, float16 or bfloat16")
    return code


def _all_here(dtype, *tensors) -> bool:
    """Whether all are tensors of `dtype` on the current device: the common case, asked at once."""
    try:
        index = tensors[0].get_device()   # -1 of a host tensor
        for t in tensors:
            if t.get_device() != index or t.dtype is not dtype:
                return False
    except AttributeError:   # no tensor
        return False
    return index >= 0 and index == torch._C._cuda_getDevice()


def _stream() -> int:
    """The current stream of the current device (torch.cuda.current_stream().cuda_stream without the object around it: 2 us less)."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _written(t) -> None:
    """Tells autograd that `t` was changed in place, so that a backward pass which needs its old values refuses."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _differentiated(*tensors) -> bool:
    """Whether a call goes through autograd: one of these needs a gradient, or forward-mode derivatives are being taken.  A tensor that
    carries such a derivative does not need a gradient and has an ordinary pointer; autograd refuses it, as the operators have none."""
    return torch.autograd.forward_ad._current_level >= 0 or torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


# An allocation without torch's dispatch of it, where torch has one of this signature: 0.8 us instead of 1.7, of calls that take 8.  Through torch where something
# looks at what is dispatched (a mode that counts memory, say) or fills new memory (deterministic algorithms).
_EMPTY_STRIDED = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)
_DISPATCH_MODES = getattr(torch._C, "_len_torch_dispatch_stack", None)
_DETERMINISTIC = getattr(torch._C, "_get_deterministic_algorithms", torch.are_deterministic_algorithms_enabled)


def _dispatched(shape, dtype):
    return torch.empty(shape, device="cuda", dtype=dtype)


def _direct(shape, dtype):
    global _EMPTY_STRIDED
    if 0 in shape:
        return _dispatched(shape, dtype)
    try:
        if len(shape) == 2:
            return _EMPTY_STRIDED(tuple(shape), (shape[1], 1), dtype)
        strides, stride = [], 1
        for n in reversed(shape):
            strides.append(stride)
            stride *= n
        return _EMPTY_STRIDED(tuple(shape), tuple(reversed(strides)), dtype)
    except TypeError:   # another signature, or none
        _EMPTY_STRIDED = None
        return _dispatched(shape, dtype)


def _allocation():
    """What allocates a call's tensors: (shape, dtype) -> a contiguous tensor on the current device, of any content."""
    return _dispatched if _EMPTY_STRIDED is None or _DISPATCH_MODES is None or _DISPATCH_MODES() or _DETERMINISTIC() else _direct


def _scratch(size: int, empty):
    """`size` bytes on the current device, None where there are to be none."""
    return empty((size,), torch.uint8) if size else None


# ---- layer norm

def _rows(t):
    """`t` as (rows, width) with contiguous rows; a copy only where its layout has no such view."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check_parameter(name: str, t, width: int) -> None:
    if t is not None:
        if not _all_here(torch.float32, t):
            _device_tensor(name, t, torch.float32)
        if t.shape != (width,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of shape ({width},)")


def layer_norm_forward(x, weight=None, bias=None, *, eps: float = 1e-5, residual=None) -> Tuple:
    """total = x + residual (rounded to x's type; x itself without a residual), and the layer norm of it over the last axis.

    x, residual (..., width) float32 / float16 / bfloat16; weight, bias (width,) float32 or None.
    Returns (y, total, mean, rstd): y and total of x's shape and type, mean and rstd (rows,) float32, which
    layer_norm_backward takes."""
    code = _device_tensor("x", x)
    shape = x.shape
    if not shape:
        raise ValueError("x must have a last axis to normalise over")
    width = shape[-1]
    if residual is not None:
        _device_tensor("residual", residual, x.dtype)
        if residual.shape != shape:
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
    y = torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, device=x.device, dtype=x.dtype)
    total = x if residual is None else torch.empty_like(y)
    mean, rstd = torch.empty((2, rows), device=x.device, dtype=torch.float32).unbind(0)
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
    @once_differentiable
    def backward(ctx, dy, d_total):
        total, weight, mean, rstd = ctx.saved_tensors
        if dy is None:
            return d_total, d_total, None, None, None
        dx, dweight, dbias = layer_norm_backward(dy, total, weight, mean, rstd, d_total=d_total, want_parameters=ctx.wanted)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dx if need[1] else None, dweight if need[2] else None, dbias if need[3] else None, None


def layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5, residual=None):
    """layer_norm_forward with autograd: y, or with a residual (y, total)."""
    if _differentiated(x, residual, weight, bias):
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


# ---- attention with a decaying state

# flstm_rows and flstm_decay_attention, packed: a call of a few microseconds has no time for ctypes structures
_ROWS = struct.Struct("@Pnnn")
_SHAPE = struct.Struct("@NNPiiiiifP")


def _rows_of(t):
    """Where (sequences, tokens, heads, D) or, packed, (tokens, heads, D) lies; for a single token (sequences, heads, D) too, where the
    token's stride is not read."""
    if t is None:
        return None
    s = t.stride()
    return _ROWS.pack(t.data_ptr(), s[0], s[-3], s[-2])


def _last_axis_contiguous(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _tokens_within_reach(t):
    """The kernels form the offsets of a chunk's tokens in 32 bits, for distances below 2^23 elements: tensors with more between two tokens
    (a transposed (tokens, sequences, ..) of very many features) are copied, sequence by sequence."""
    return t.contiguous() if t.shape[-3] > 1 and t.stride(-3) >= 1 << 23 else t


def _decay_shape(q, k, v, log_decay, scale, state, cu_seqlens, axes: int):
    """Checks q (.., heads, dk), k (.., kv_heads, dk) and v (.., kv_heads, dv) of `axes` axes, and what goes with them."""
    if not (_all_here(torch.float32, log_decay) and isinstance(q, torch.Tensor) and q.dtype in _DTYPES and _all_here(q.dtype, q, k, v)):
        _device_tensor("q", q)
        for name, t in (("k", k), ("v", v)):
            _device_tensor(name, t, q.dtype)
        _device_tensor("log_decay", log_decay, torch.float32)
    code, of_q, of_k, of_v = _DTYPES[q.dtype], q.shape, k.shape, v.shape
    if len(of_q) != axes:
        raise ValueError(f"q must have {axes} axes, not {len(of_q)}")
    heads, dk = of_q[-2:]
    for name, shape in (("k", of_k), ("v", of_v)):
        if len(shape) != axes or shape[:-2] != of_q[:-2]:
            raise ValueError(f"{name} must have q's leading axes {tuple(of_q[:-2])}: got {tuple(shape)}")
    kv_heads, dv = of_v[-2:]
    if of_k[-2:] != (kv_heads, dk):
        raise ValueError(f"k must have v's heads and q's width ({kv_heads}, {dk}): got {tuple(of_k[-2:])}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads != 0:
        raise ValueError(f"the number of query heads ({heads}) must be a multiple of that of key and value heads ({kv_heads})")
    if not (8 <= dk <= 256 and 8 <= dv <= 256):
        raise ValueError(f"head widths must lie in 8 .. 256: got {dk} and {dv}")
    if log_decay.shape != (heads,) or not log_decay.is_contiguous():
        raise ValueError(f"log_decay must be a contiguous tensor of shape ({heads},)")
    if log_decay.requires_grad:
        raise ValueError("log_decay is a constant of the model: it has no gradient")
    scale = dk ** -0.5 if scale is None else float(scale)
    if scale != scale:
        raise ValueError("scale must be a number")
    if cu_seqlens is not None:
        _device_tensor_int("cu_seqlens", cu_seqlens)
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1 or not cu_seqlens.is_contiguous():
            raise ValueError("cu_seqlens must be a contiguous tensor of one more entry than there are sequences")
        sequences, tokens = cu_seqlens.shape[0] - 1, of_q[0]
    else:
        sequences, tokens = of_q[0], of_q[1] if axes == 4 else 1
    shape = _SHAPE.pack(sequences, tokens, _ptr(cu_seqlens) or 0, heads, kv_heads, dk, dv, code, scale, log_decay.data_ptr())
    _check_state("state", state, (sequences, heads, dk, dv))
    return shape, (sequences, heads, dk, dv)


def _device_tensor_int(name: str, t) -> None:
    if not torch.is_tensor(t) or not t.is_cuda or t.get_device() != torch.cuda.current_device():
        raise ValueError(f"{name} must be a CUDA tensor on the current device")
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be of type {torch.int32}, not {t.dtype}")


def _check_state(name: str, t, shape) -> None:
    if t is not None:
        if not _all_here(torch.float32, t):
            _device_tensor(name, t, torch.float32)
        if t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of shape {shape}")


def _like_rows(q, heads: int, width: int):
    """An output in the memory order of q's rows: (T, B, ..) below a transposed (B, T, ..) stays that."""
    if q.dim() == 4 and q.stride(0) < q.stride(1) and q.shape[0] > 1:
        return torch.empty((q.shape[1], q.shape[0], heads, width), device=q.device, dtype=q.dtype).transpose(0, 1)
    return torch.empty((*q.shape[:-2], heads, width), device=q.device, dtype=q.dtype)


def _workspace(shape: bytes, backward: int, device):
    size = _bind().flstm_decay_attention_workspace_bytes(shape, backward)
    return torch.empty(size, device=device, dtype=torch.uint8) if size else None


def decay_attention_forward(q, k, v, log_decay, *, scale: Optional[float] = None, state=None, cu_seqlens=None,
                            want_state: bool = True) -> Tuple:
    """S_t = exp(log_decay) S_{t-1} + k_t v_t^T, o_t = scale * S_t^T q_t, for every sequence and head.

    q (sequences, tokens, heads, dk), k (.., kv_heads, dk), v (.., kv_heads, dv), float32 / float16 / bfloat16, of any strides
    (a transposed (tokens, sequences, ..) among them); head h reads key and value head h // (heads // kv_heads).  Or packed,
    (tokens, heads, dk) and so on, with cu_seqlens (sequences + 1,) int32, from 0 on.  log_decay (heads,) float32, <= 0, a constant.
    scale: dk ** -0.5 where None.  state (sequences, heads, dk, dv) float32: the state in front of the first tokens (None: zeros).
    Returns (o, state behind the last tokens or, without want_state, None)."""
    axes = 4 if cu_seqlens is None else 3
    shape, states = _decay_shape(q, k, v, log_decay, scale, state, cu_seqlens, axes)
    q, k, v = (_last_axis_contiguous(t) for t in (q, k, v))
    o = _like_rows(q, states[1], states[3])
    q, k, v = (_tokens_within_reach(t) for t in (q, k, v))
    final = torch.empty(states, device=q.device, dtype=torch.float32) if want_state else None
    workspace = _workspace(shape, 0, q.device)
    _check(_bind().flstm_decay_attention_forward(shape, _rows_of(q), _rows_of(k), _rows_of(v), _ptr(state), _rows_of(o),
                                                 _ptr(final), _ptr(workspace), _stream()), "flstm_decay_attention_forward")
    return o, final


def decay_attention_backward(do, q, k, v, log_decay, *, scale: Optional[float] = None, state=None, cu_seqlens=None, d_state=None,
                             want=(True, True, True, True)) -> Tuple:
    """Gradients (dq, dk, dv, d_initial_state) of decay_attention_forward from those of o and of the final state (None: zeros);
    `want` tells which (None for the others)."""
    axes = 4 if cu_seqlens is None else 3
    shape, states = _decay_shape(q, k, v, log_decay, scale, state, cu_seqlens, axes)
    _device_tensor("do", do, q.dtype)
    if tuple(do.shape) != (*q.shape[:-1], states[3]):
        raise ValueError(f"do must have shape {(*q.shape[:-1], states[3])}: got {tuple(do.shape)}")
    _check_state("d_state", d_state, states)
    do, q, k, v = (_last_axis_contiguous(t) for t in (do, q, k, v))
    dq = _like_rows(q, *q.shape[-2:]) if want[0] else None
    dk = _like_rows(k, *k.shape[-2:]) if want[1] else None
    dv = _like_rows(v, *v.shape[-2:]) if want[2] else None
    do, q, k, v = (_tokens_within_reach(t) for t in (do, q, k, v))
    d_initial = torch.empty(states, device=q.device, dtype=torch.float32) if want[3] else None
    workspace = _workspace(shape, 1, q.device)
    _check(_bind().flstm_decay_attention_backward(
        shape, _rows_of(do), _rows_of(q), _rows_of(k), _rows_of(v), _ptr(state), _ptr(d_state), _rows_of(dq), _rows_of(dk),
        _rows_of(dv), _ptr(d_initial), _ptr(workspace), _stream()), "flstm_decay_attention_backward")
    return dq, dk, dv, d_initial


def decay_attention_step(q, k, v, log_decay, state, *, scale: Optional[float] = None):
    """One token of every sequence: q (sequences, heads, dk), k (sequences, kv_heads, dk), v (sequences, kv_heads, dv); `state`
    (sequences, heads, dk, dv) float32 is updated in place.  Returns o (sequences, heads, dv).  No autograd."""
    if state is None:
        raise ValueError("state must be a tensor: it is updated in place")
    shape, states = _decay_shape(q, k, v, log_decay, scale, state, None, 3)
    q, k, v = (_last_axis_contiguous(t) for t in (q, k, v))
    o = torch.empty_like(q) if states[2] == states[3] and q.is_contiguous() else torch.empty((states[0], states[1], states[3]), device=q.device, dtype=q.dtype)
    _check(_bind().flstm_decay_attention_step(shape, _rows_of(q), _rows_of(k), _rows_of(v), _rows_of(o), state.data_ptr(),
                                              _stream()), "flstm_decay_attention_step")
    _written(state)
    return o


class _DecayAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, state, log_decay, scale, cu_seqlens):
        o, final = decay_attention_forward(q, k, v, log_decay, scale=scale, state=state, cu_seqlens=cu_seqlens)
        ctx.save_for_backward(q, k, v, state, log_decay, cu_seqlens)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    @once_differentiable
    def backward(ctx, do, d_final):
        q, k, v, state, log_decay, cu_seqlens = ctx.saved_tensors
        if do is None:
            do = torch.zeros((*q.shape[:-1], v.shape[-1]), device=q.device, dtype=q.dtype)
        if d_final is not None:
            d_final = d_final.contiguous()
        grads = decay_attention_backward(do, q, k, v, log_decay, scale=ctx.scale, state=state, cu_seqlens=cu_seqlens, d_state=d_final,
                                         want=ctx.needs_input_grad[:4])
        return (*grads, None, None, None)


def decay_attention(q, k, v, log_decay, *, scale: Optional[float] = None, state=None, cu_seqlens=None) -> Tuple:
    """decay_attention_forward with autograd in q, k, v and state: (o, final state)."""
    if _differentiated(q, k, v, state):
        return _DecayAttentionFunction.apply(q, k, v, state, log_decay, scale, cu_seqlens)
    return decay_attention_forward(q, k, v, log_decay, scale=scale, state=state, cu_seqlens=cu_seqlens)


# ---- distillation from a teacher's top logits

_PROBLEM = struct.Struct("@NNPNiiPiPif")   # flstm_distillation


def _distillation(logits, teacher_logits, teacher_index, temperature: float):
    """The checked problem and the tensors that it points into, which the caller keeps until its call is enqueued."""
    code = _device_tensor("logits", logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must have a last axis of at least one entry")
    teacher_code = _device_tensor("teacher_logits", teacher_logits)
    if not torch.is_tensor(teacher_index) or not teacher_index.is_cuda or teacher_index.get_device() != logits.get_device():
        raise ValueError("teacher_index must be a CUDA tensor on the device of logits")
    if teacher_index.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"teacher_index must be of type int32 or int64, not {teacher_index.dtype}")
    if teacher_logits.shape != teacher_index.shape or teacher_logits.shape[:-1] != logits.shape[:-1] or teacher_logits.dim() != logits.dim():
        raise ValueError(f"teacher_logits and teacher_index must have shape {(*logits.shape[:-1], 'top')}: got {tuple(teacher_logits.shape)} "
                         f"and {tuple(teacher_index.shape)}")
    top = teacher_logits.shape[-1]
    if not 1 <= top <= 1024:
        raise ValueError(f"between 1 and 1024 teacher entries a row: got {top}")
    temperature = float(temperature)
    if not 0 < temperature < float("inf"):
        raise ValueError("temperature must be a positive number")
    rows, vocabulary = logits.shape[:-1].numel(), logits.shape[-1]
    kept = (_rows(logits) if rows else logits, teacher_logits.contiguous(), teacher_index.contiguous())
    # (rows that share memory, an expanded tensor, are told apart by nothing but their number)
    ld = kept[0].stride(0) if rows > 1 else vocabulary
    if ld < vocabulary:
        kept = (kept[0].contiguous(), *kept[1:])
        ld = vocabulary
    problem = _PROBLEM.pack(rows, vocabulary, kept[0].data_ptr(), ld, code, top, kept[1].data_ptr(), teacher_code, kept[2].data_ptr(),
                            teacher_index.dtype == torch.int64, temperature)
    return problem, rows, vocabulary, ld, kept


def _per_row(name: str, t, rows: int):
    """`t` as (rows,) float32 with any stride (0: one value for all rows)."""
    _device_tensor(name, t, torch.float32)
    if t.numel() == 1 and rows != 1:
        return t.reshape(1).expand(rows)
    if t.numel() != rows:
        raise ValueError(f"{name} must hold one value a row ({rows}) or one for all: got {t.numel()}")
    return t if t.dim() == 1 else t.reshape(-1)


def distillation_forward(logits, teacher_logits, teacher_index, *, temperature: float = 1.0) -> Tuple:
    """temperature^2 KL(p || q) for every row, p = softmax(teacher_logits / temperature) over the row's entries and
    q = softmax(logits / temperature) over the vocabulary.

    logits (.., vocabulary), teacher_logits (.., top) float32 / float16 / bfloat16, teacher_index (.., top) int32 / int64.  Entries
    with an index outside the vocabulary (-1, say) or a logit of minus infinity do not count; a row without others has loss 0.
    Returns (loss, stats), float32: loss of logits' leading shape, stats (rows, 2), which distillation_backward takes (a row's
    largest logit, and log2 of the sum of exp((logit - largest) / temperature))."""
    problem, rows, vocabulary, ld, kept = _distillation(logits, teacher_logits, teacher_index, temperature)
    loss = torch.empty(logits.shape[:-1], device=logits.device, dtype=torch.float32)
    stats = torch.empty((rows, 2), device=logits.device, dtype=torch.float32)
    _check(_bind().flstm_distillation_forward(problem, loss.data_ptr(), stats.data_ptr(), _stream()), "flstm_distillation_forward")
    return loss, stats


def distillation_backward(d_loss, logits, teacher_logits, teacher_index, stats, *, temperature: float = 1.0):
    """The gradient of logits (in their type) from that of every row's loss (one value a row, or one for all)."""
    problem, rows, vocabulary, ld, kept = _distillation(logits, teacher_logits, teacher_index, temperature)
    d_loss = _per_row("d_loss", d_loss, rows)
    _device_tensor("stats", stats, torch.float32)
    if tuple(stats.shape) != (rows, 2) or not stats.is_contiguous():
        raise ValueError(f"stats must be a contiguous tensor of shape ({rows}, 2)")
    dlogits = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
    _check(_bind().flstm_distillation_backward(problem, stats.data_ptr(), d_loss.data_ptr(), d_loss.stride(0) if rows else 0,
                                               dlogits.data_ptr(), vocabulary, _stream()), "flstm_distillation_backward")
    return dlogits


def distillation_train(logits, teacher_logits, teacher_index, d_loss, *, temperature: float = 1.0, in_place: bool = False) -> Tuple:
    """(loss, dlogits) in one call, for a d_loss that is known beforehand (1 / rows for a mean): the logits are read once.
    in_place: the gradient takes the place of the logits, which must then have contiguous rows."""
    problem, rows, vocabulary, ld, kept = _distillation(logits, teacher_logits, teacher_index, temperature)
    d_loss = _per_row("d_loss", d_loss, rows)
    if in_place and rows and kept[0].data_ptr() != logits.data_ptr():
        raise ValueError("in place, logits must have contiguous rows of their own")
    loss = torch.empty(logits.shape[:-1], device=logits.device, dtype=torch.float32)
    dlogits = logits if in_place else torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
    lib = _bind()
    size = lib.flstm_distillation_workspace_bytes(problem)
    workspace = torch.empty(size, device=logits.device, dtype=torch.uint8) if size else None
    _check(lib.flstm_distillation_train(problem, d_loss.data_ptr(), d_loss.stride(0) if rows else 0, loss.data_ptr(),
                                        dlogits.data_ptr(), ld if in_place else vocabulary, _ptr(workspace), _stream()),
           "flstm_distillation_train")
    if in_place:
        _written(logits)
    return loss, dlogits


class _DistillationFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_index, temperature):
        loss, stats = distillation_forward(logits, teacher_logits, teacher_index, temperature=temperature)
        ctx.save_for_backward(logits, teacher_logits, teacher_index, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss):
        logits, teacher_logits, teacher_index, stats = ctx.saved_tensors
        return distillation_backward(d_loss, logits, teacher_logits, teacher_index, stats, temperature=ctx.temperature), None, None, None


def distillation_loss(logits, teacher_logits, teacher_index, *, temperature: float = 1.0):
    """distillation_forward's loss of every row, with autograd in logits (the teacher gets no gradient)."""
    if _differentiated(logits):
        return _DistillationFunction.apply(logits, teacher_logits, teacher_index, temperature)
    return distillation_forward(logits, teacher_logits, teacher_index, temperature=temperature)[0]


# ---- embedding of tokens

_EMBEDDING = struct.Struct("@NNNPif0P")   # flstm_embedding


def _indices(name: str, t) -> bool:
    """Refuses what holds no int32 or int64 on the current device; returns whether it is int64."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"{name} must be a CUDA tensor on the current device")
    kind = t.dtype
    if kind is not torch.int64 and kind is not torch.int32:
        raise ValueError(f"{name} must be of type int32 or int64, not {kind}")
    return kind is torch.int64


def _op_dtype(name: str, dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"unsupported {name} {dtype}: it must be float32, float16 or bfloat16")
    return code


def _scale(scale) -> float:
    scale = float(scale)
    if not abs(scale) <= 3.4028234663852886e38:
        raise ValueError("scale must be a finite number")
    return scale


def embedding_forward(tokens, table, *, scale: float = 1.0, dtype=None):
    """out[..., :] = scale * table[tokens[...]], rounded once to `dtype` (table's where None); zeros for a token outside the vocabulary (-1,
    say).

    tokens int32 / int64 of any shape, table (vocabulary, width) float32 / float16 / bfloat16.  Returns (*tokens.shape, width)."""
    index_64, code = _indices("tokens", tokens), _device_tensor("table", table)
    if table.dim() != 2 or table.shape[0] < 1:
        raise ValueError(f"table must have shape (vocabulary, width): got {tuple(table.shape)}")
    dtype = table.dtype if dtype is None else dtype
    out_code, scale = _op_dtype("dtype", dtype), _scale(scale)
    (vocabulary, width), tokens = table.shape, tokens.contiguous()
    out = _allocation()((*tokens.shape, width), dtype)
    if out.numel() == 0:
        return out
    rows, ld = table, width
    if not table.is_contiguous():
        rows = _rows(table)
        if rows.stride(0) < width and vocabulary > 1:   # (rows that share memory)
            rows = rows.contiguous()
        ld = rows.stride(0)
    problem = _EMBEDDING.pack(tokens.numel(), vocabulary, width, tokens.data_ptr(), index_64, scale)
    _check(_bind().flstm_embedding_forward(problem, rows.data_ptr(), ld, code, out.data_ptr(), out_code, _stream()),
           "flstm_embedding_forward")
    return out


def embedding_backward(d_out, tokens, vocabulary: int, *, scale: float = 1.0, dtype=torch.float32):
    """The table's gradient (vocabulary, width) of type `dtype` from that of embedding_forward's result, d_out (*tokens.shape, width): for each
    token scale times the sum of its rows, zeros for tokens that do not occur."""
    index_64, code = _indices("tokens", tokens), _device_tensor("d_out", d_out)
    if d_out.dim() != tokens.dim() + 1 or d_out.shape[:-1] != tokens.shape:
        raise ValueError(f"d_out must have shape {(*tokens.shape, 'width')}: got {tuple(d_out.shape)}")
    if vocabulary < 1:
        raise ValueError("vocabulary must be >= 1")
    out_code, scale, width = _op_dtype("dtype", dtype), _scale(scale), d_out.shape[-1]
    empty = _allocation()
    d_table = empty((vocabulary, width), dtype)
    if width == 0:
        return d_table
    tokens = tokens.contiguous()
    rows = _rows(d_out) if d_out.numel() else d_out.reshape(0, width)
    problem = _EMBEDDING.pack(tokens.numel(), vocabulary, width, tokens.data_ptr(), index_64, scale)
    lib = _bind()
    workspace = _scratch(lib.flstm_embedding_workspace_bytes(problem), empty)
    _check(lib.flstm_embedding_backward(problem, rows.data_ptr(), rows.stride(0), code, d_table.data_ptr(), out_code, _ptr(workspace), _stream()),
           "flstm_embedding_backward")
    return d_table


class _EmbeddingFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, dtype):
        ctx.save_for_backward(tokens)
        ctx.vocabulary, ctx.scale, ctx.dtype = table.shape[0], scale, table.dtype
        return embedding_forward(tokens, table, scale=scale, dtype=dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        tokens, = ctx.saved_tensors
        return embedding_backward(d_out, tokens, ctx.vocabulary, scale=ctx.scale, dtype=ctx.dtype), None, None, None


def embedding(tokens, table, *, scale: float = 1.0, dtype=None):
    """embedding_forward with autograd in table."""
    if _differentiated(table):
        return _EmbeddingFunction.apply(table, tokens, scale, dtype)
    return embedding_forward(tokens, table, scale=scale, dtype=dtype)


class Embedding(torch.nn.Module):
    """Rows of a table of fp32 parameters, named and initialised as torch.nn.Embedding's, scaled, as activations of type `dtype`; zeros for tokens outside
    the vocabulary, which are what pads (none of those inside does)."""

    padding_idx = None

    def __init__(self, vocabulary: int, width: int, *, scale: float = 1.0, dtype=torch.float32, device="cuda"):
        super().__init__()
        if vocabulary < 1 or width < 1:
            raise ValueError("vocabulary and width must be >= 1")
        _op_dtype("dtype", dtype)
        self.vocabulary, self.width, self.scale, self.dtype = int(vocabulary), int(width), _scale(scale), dtype
        self.weight = torch.nn.Parameter(torch.empty((self.vocabulary, self.width), device=device, dtype=torch.float32))
        torch.nn.init.normal_(self.weight)

    @property
    def num_embeddings(self) -> int:
        return self.vocabulary

    @property
    def embedding_dim(self) -> int:
        return self.width

    def forward(self, tokens):
        return embedding(tokens, self.weight, scale=self.scale, dtype=self.dtype)


# ---- gated linear recurrence

_RECURRENCE = struct.Struct("@NNPNi0P")   # flstm_recurrence


def _recurrence(x, forget, gate, state, cu_seqlens, axes: int):
    """Checks x, forget and gate (or None) of `axes` axes, the last of them the channels, and what goes with them."""
    tensors = (x, forget) if gate is None else (x, forget, gate)
    if not (isinstance(x, torch.Tensor) and x.dtype in _DTYPES and _all_here(x.dtype, *tensors)):
        _device_tensor("x", x)
        for name, t in (("forget", forget), ("gate", gate)):
            if t is not None:
                _device_tensor(name, t, x.dtype)
    shape = x.shape
    if len(shape) != axes:
        raise ValueError(f"x must have {axes} axes, not {len(shape)}")
    if forget.shape != shape:
        raise ValueError(f"forget must have x's shape {tuple(shape)}: got {tuple(forget.shape)}")
    if gate is not None and gate.shape != shape:
        raise ValueError(f"gate must have x's shape {tuple(shape)}: got {tuple(gate.shape)}")
    if cu_seqlens is not None:
        _device_tensor_int("cu_seqlens", cu_seqlens)
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1 or not cu_seqlens.is_contiguous():
            raise ValueError("cu_seqlens must be a contiguous tensor of one more entry than there are sequences")
        sequences, tokens = cu_seqlens.shape[0] - 1, shape[0]
    else:
        sequences, tokens = shape[0], shape[1] if axes == 3 else 1
    states = (sequences, shape[-1])
    _check_state("state", state, states)
    return _RECURRENCE.pack(sequences, tokens, _ptr(cu_seqlens) or 0, shape[-1], _DTYPES[x.dtype]), states


def _channel_rows(t, packed: bool = False):
    """Where (sequences, tokens, width), packed (tokens, width), or for a single token (sequences, width), lies."""
    if t is None:
        return None
    s = t.stride()
    return _ROWS.pack(t.data_ptr(), 0 if packed else s[0], s[-2] if packed or len(s) == 3 else 0, 0)


def _like_channels(x, empty):
    """An output in the memory order of x's rows."""
    if x.dim() == 3 and x.stride(0) < x.stride(1) and x.shape[0] > 1:
        return empty((x.shape[1], x.shape[0], x.shape[2]), x.dtype).transpose(0, 1)
    return empty(x.shape, x.dtype)


def _recurrence_workspace(shape: bytes, backward: int, empty):
    return _scratch(_bind().flstm_gated_recurrence_workspace_bytes(shape, backward), empty)


def gated_recurrence_forward(x, forget, gate=None, *, state=None, cu_seqlens=None, want_state: bool = True, want_saved: bool = True) -> Tuple:
    """c_t = f_t c_{t-1} + (1 - f_t) x_t with f = sigmoid(forget), y_t = c_t or, with a gate, sigmoid(gate_t) c_t, for every channel of every sequence.

    x, forget, gate (sequences, tokens, width) float32 / float16 / bfloat16, of any strides (parts of one projection, a transposed
    (tokens, sequences, width)).  Or packed, (tokens, width), with cu_seqlens (sequences + 1,) int32, from 0 on.  state (sequences, width)
    float32: the state in front of the first tokens (None: zeros).
    Returns (y, state behind the last tokens, saved), the latter two None where not wanted; gated_recurrence_backward takes saved."""
    packed = cu_seqlens is not None
    shape, states = _recurrence(x, forget, gate, state, cu_seqlens, 2 if packed else 3)
    x, forget = _last_axis_contiguous(x), _last_axis_contiguous(forget)
    gate = None if gate is None else _last_axis_contiguous(gate)
    empty, lib = _allocation(), _bind()
    y = _like_channels(x, empty)
    final = empty(states, torch.float32) if want_state else None
    saved = empty((lib.flstm_gated_recurrence_saved_rows(shape), states[1]), torch.float32) if want_saved else None
    workspace = _recurrence_workspace(shape, 0, empty)
    _check(lib.flstm_gated_recurrence_forward(shape, _channel_rows(x, packed), _channel_rows(forget, packed), _channel_rows(gate, packed), _ptr(state),
                                              _channel_rows(y, packed), _ptr(final), _ptr(saved), _ptr(workspace), _stream()),
           "flstm_gated_recurrence_forward")
    return y, final, saved


def gated_recurrence_backward(dy, x, forget, gate, saved, *, d_state=None, cu_seqlens=None, want=(True, True, True, True)) -> Tuple:
    """Gradients (dx, dforget, dgate, d_initial_state) of gated_recurrence_forward from those of y and of the final state (None: zeros); `want`
    tells which (None for the others, and for dgate without a gate).  saved: what the forward pass returned."""
    packed = cu_seqlens is not None
    shape, states = _recurrence(x, forget, gate, d_state, cu_seqlens, 2 if packed else 3)
    _device_tensor("dy", dy, x.dtype)
    if dy.shape != x.shape:
        raise ValueError(f"dy must have x's shape {tuple(x.shape)}: got {tuple(dy.shape)}")
    lib = _bind()
    _check_state("saved", saved, (lib.flstm_gated_recurrence_saved_rows(shape), states[1]))
    if saved is None:
        raise ValueError("saved must be what the forward pass returned")
    dy, x, forget = (_last_axis_contiguous(t) for t in (dy, x, forget))
    gate = None if gate is None else _last_axis_contiguous(gate)
    empty = _allocation()
    dx = _like_channels(x, empty) if want[0] else None
    dforget = _like_channels(x, empty) if want[1] else None
    dgate = _like_channels(x, empty) if want[2] and gate is not None else None
    d_initial = empty(states, torch.float32) if want[3] else None
    workspace = _recurrence_workspace(shape, 1, empty)
    _check(lib.flstm_gated_recurrence_backward(
        shape, _channel_rows(dy, packed), _channel_rows(x, packed), _channel_rows(forget, packed), _channel_rows(gate, packed), saved.data_ptr(),
        _ptr(d_state), _channel_rows(dx, packed), _channel_rows(dforget, packed), _channel_rows(dgate, packed), _ptr(d_initial), _ptr(workspace),
        _stream()), "flstm_gated_recurrence_backward")
    return dx, dforget, dgate, d_initial


def gated_recurrence_step(x, forget, state, gate=None):
    """One token of every sequence: x, forget, gate (sequences, width); `state` (sequences, width) float32 is updated in place.  Returns y.
    No autograd."""
    if state is None:
        raise ValueError("state must be a tensor: it is updated in place")
    shape, states = _recurrence(x, forget, gate, state, None, 2)
    x, forget = _last_axis_contiguous(x), _last_axis_contiguous(forget)
    gate = None if gate is None else _last_axis_contiguous(gate)
    y = _allocation()(states, x.dtype)
    _check(_bind().flstm_gated_recurrence_step(shape, _channel_rows(x), _channel_rows(forget), _channel_rows(gate), _channel_rows(y), state.data_ptr(),
                                               _stream()), "flstm_gated_recurrence_step")
    _written(state)
    return y


class _GatedRecurrenceFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, forget, gate, state, cu_seqlens):
        y, final, saved = gated_recurrence_forward(x, forget, gate, state=state, cu_seqlens=cu_seqlens)
        ctx.save_for_backward(x, forget, gate, saved, cu_seqlens)
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, d_final):
        x, forget, gate, saved, cu_seqlens = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros(x.shape, device=x.device, dtype=x.dtype)
        if d_final is not None:
            d_final = d_final.contiguous()
        grads = gated_recurrence_backward(dy, x, forget, gate, saved, d_state=d_final, cu_seqlens=cu_seqlens, want=ctx.needs_input_grad[:4])
        return (*grads, None)


def gated_recurrence(x, forget, gate=None, *, state=None, cu_seqlens=None) -> Tuple:
    """gated_recurrence_forward with autograd in x, forget, gate and state: (y, final state)."""
    if _differentiated(x, forget, gate, state):
        return _GatedRecurrenceFunction.apply(x, forget, gate, state, cu_seqlens)
    return gated_recurrence_forward(x, forget, gate, state=state, cu_seqlens=cu_seqlens, want_saved=False)[:2]


# ---- beam search

_BEAMS = struct.Struct("@NiiNPNiPPq")   # flstm_beams
_BEAM_STATE = struct.Struct("@PNN")
_MAX_BEAMS = 32


def beam_select(logits, scores, *, beams: Optional[int] = None, end: Optional[int] = None, finished=None) -> Tuple:
    """The best continuations of every sequence's hypotheses by one token, by scores + log_softmax(logits), the best first and of equal ones
    that of the lower hypothesis and token.  (The sum in log_softmax is held in 32 bits: continuations of different hypotheses that are nearer than 48 * 2^-24
    may come in either order, unless logits and scores are equal.)

    logits (sequences, hypotheses, vocabulary) float32 / float16 / bfloat16, scores (sequences, hypotheses) float32 (minus infinity: no
    hypothesis).  beams: how many are kept, as many as there are where None; up to 32 of both.  end: the token that ends a hypothesis;
    finished (sequences, hypotheses) bool: those that are, which stay as they are, with `end` as their token.
    Returns (scores, parents, tokens, finished), (sequences, beams) of float32, int64, int64 and bool (None without `end`).  Logits of minus
    infinity and NaN are no continuations; where there are too few, scores are minus infinity and tokens -1.  No autograd."""
    code, of = _device_tensor("logits", logits), logits.shape
    if len(of) != 3 or of[2] < 1:
        raise ValueError(f"logits must have shape (sequences, hypotheses, vocabulary): got {tuple(of)}")
    sequences, hypotheses, vocabulary = of
    keep = hypotheses if beams is None else int(beams)
    if not (1 <= hypotheses <= _MAX_BEAMS and 1 <= keep <= _MAX_BEAMS):
        raise ValueError(f"between 1 and {_MAX_BEAMS} hypotheses and beams: got {hypotheses} and {keep}")
    if not _all_here(torch.float32, scores):
        _device_tensor("scores", scores, torch.float32)
    if scores.shape != (sequences, hypotheses):
        raise ValueError(f"scores must have shape {(sequences, hypotheses)}: got {tuple(scores.shape)}")
    if end is not None and not 0 <= end < vocabulary:
        raise ValueError(f"end must lie in the vocabulary: got {end}")
    if finished is not None:
        if end is None:
            raise ValueError("finished hypotheses need an `end`")
        if not _all_here(torch.bool, finished):
            raise ValueError("finished must be a bool tensor on the device of logits")
        if finished.shape != (sequences, hypotheses):
            raise ValueError(f"finished must have shape {(sequences, hypotheses)}: got {tuple(finished.shape)}")
        finished = finished.contiguous()
    scores = scores.contiguous()
    rows, ld = logits, vocabulary
    if not logits.is_contiguous():
        rows = _rows(logits)
        ld = rows.stride(0) if sequences * hypotheses > 1 else vocabulary
        if ld < vocabulary:   # (rows that share memory)
            rows, ld = rows.contiguous(), vocabulary
    shape = (sequences, keep)
    empty = _allocation()
    out_scores, parents, tokens = empty(shape, torch.float32), empty(shape, torch.int64), empty(shape, torch.int64)
    out_finished = None if end is None else empty(shape, torch.bool)
    problem = _BEAMS.pack(sequences, hypotheses, keep, vocabulary, rows.data_ptr(), ld, code, scores.data_ptr(), _ptr(finished) or 0,
                          -1 if end is None else end)
    lib = _bind()
    workspace = _scratch(lib.flstm_beam_select_workspace_bytes(problem), empty)
    _check(lib.flstm_beam_select(problem, out_scores.data_ptr(), parents.data_ptr(), tokens.data_ptr(), _ptr(out_finished), _ptr(workspace),
                                 _stream()), "flstm_beam_select")
    return out_scores, parents, tokens, out_finished


def beam_reorder(parents, *states) -> None:
    """Hypothesis b of sequence s becomes, in every one of `states`, what hypothesis parents[s, b] was, in place; rows that stay are not touched.

    parents (sequences, hypotheses) int64, as beam_select returns them; up to 32 hypotheses; one outside them leaves its row as it is.  states: tensors
    of any type, (sequences * hypotheses, ..) or (sequences, hypotheses, ..), with contiguous rows, that share no memory.  No autograd."""
    if not torch.is_tensor(parents) or not parents.is_cuda or parents.get_device() != torch._C._cuda_getDevice() or parents.dtype != torch.int64:
        raise ValueError("parents must be an int64 CUDA tensor on the current device")
    if parents.dim() != 2 or not 1 <= parents.shape[1] <= _MAX_BEAMS:
        raise ValueError(f"parents must have shape (sequences, hypotheses), of 1 to {_MAX_BEAMS}: got {tuple(parents.shape)}")
    sequences, hypotheses = parents.shape
    rows, device, packed = sequences * hypotheses, parents.get_device(), []
    for i, t in enumerate(states):
        if not isinstance(t, torch.Tensor) or t.get_device() != device:
            raise ValueError(f"state {i} must be a CUDA tensor on the device of parents")
        of, strides = t.shape, t.stride()
        axes = 1 if of[:1] == (rows,) else 2
        if axes == 2 and not (of[:2] == (sequences, hypotheses) and (sequences == 1 or hypotheses == 1 or strides[0] == hypotheses * strides[1])):
            raise ValueError(f"state {i} must have {sequences} x {hypotheses} rows, evenly spaced: got shape {tuple(of)}")
        if rows and t.is_contiguous():
            stride = size = t.numel() // rows
        else:
            stride, size, whole = strides[0 if axes == 1 or hypotheses == 1 else 1], 1, True
            for n, s in zip(of[:axes - 1:-1], strides[:axes - 1:-1]):
                whole = whole and (n == 1 or s == size)
                size *= n
            if rows and size and (not whole or rows > 1 and stride < size):
                raise ValueError(f"state {i} must have contiguous rows of its own")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"state {i} needs a gradient: it would be changed in place")
        element = t.element_size()
        packed.append(_BEAM_STATE.pack(t.data_ptr(), max(stride, size) * element, size * element))
    parents = parents.contiguous()
    rc = _bind().flstm_beam_reorder(sequences, hypotheses, parents.data_ptr(), b"".join(packed), len(packed), _stream())
    if rc == 1:
        raise ValueError("states must not share memory, with each other or with parents: it would be moved twice")
    _check(rc, "flstm_beam_reorder")
    torch.autograd.graph.increment_version([t for t in states if not t.is_inference()])   # (as _written, of all at once)
