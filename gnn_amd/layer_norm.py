"""Layer norm over the last dimension: ``y = (x - mean) / sqrt(var + eps) * weight + bias`` per row, forward and
backward on the kernels of ``csrc/rwk_layer_norm.hip``.

The per-row companion of the head's batch norm (``rwgnn2/model.py:21,68``) for node features, walk steps and other
wide rows: float32, float16 or bfloat16 rows of any width, weights of the same type or float32.  All sums are fp32 in
a fixed order, with one rounding to the element type at the end, so results are bitwise reproducible.  HIP devices
only.
"""
from __future__ import annotations

import ctypes
from ctypes import c_float, c_int32, c_int64, c_void_p

import torch
import torch.nn as nn

from . import _lib

__all__ = ["layer_norm", "LayerNorm"]


class _Args(ctypes.Structure):
    """``rwk_layer_norm`` of ``rwk.h``."""
    _fields_ = [(n, c_void_p) for n in ("x", "weight", "bias", "y", "mean", "rstd", "dy", "dx", "partials", "dw", "db")] \
        + [(n, c_int64) for n in ("x_stride", "dy_stride", "rows", "width")] \
        + [("type", c_int32), ("weight_type", c_int32), ("eps", c_float)]


def _rows(t: torch.Tensor):
    """``t`` as (rows, width) with adjacent elements in a row and rows at least a width apart - a view if it can be -
    and the rows' distance in elements."""
    width = t.shape[-1]
    if t.is_contiguous():
        return t, width
    t = t.reshape(-1, width)
    if (width > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < width):
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else width


def _check(x, weight, bias):
    if not x.is_cuda:
        raise RuntimeError("gnn_amd runs on HIP devices only (no CPU fallback)")
    shape, dtype, device = x.shape, x.dtype, x.device
    _lib.element_type(dtype)
    if len(shape) < 1 or shape[-1] == 0:
        raise ValueError("x needs a last dimension of at least one")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != shape[-1:]:
            raise ValueError(f"{name} has shape {tuple(t.shape)} for rows of {shape[-1]}")
        if t.dtype is not dtype and t.dtype is not torch.float32:
            raise TypeError(f"{name} must have the type of x or float32")
        if t.device != device:
            raise RuntimeError(f"x and {name} must be on the same device")
    if bias is not None and bias.dtype is not weight.dtype:
        raise TypeError("weight and bias must have the same type")


def _forward(x, weight, bias, eps, keep):
    """(y, what the backward pass needs): x as the kernel read it, the weight, the rows' mean and 1 / deviation, the
    call's arguments."""
    rows, stride = _rows(x)
    dev, a = x.device, _Args()
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    width = x.shape[-1]
    a.x_stride, a.width, a.eps = stride, width, eps
    a.rows = n = x.numel() // width
    a.type, a.weight_type = _lib.element_type(x.dtype), _lib.element_type(weight.dtype)
    stats = None
    if keep:
        stats = torch.empty((2, n), dtype=torch.float32, device=dev)
        a.mean = at = stats.data_ptr()
        a.rstd = at + 4 * n
    if not weight.is_contiguous():
        weight = weight.contiguous()
    if n:
        if bias is not None:
            bias = bias.contiguous()
            a.bias = bias.data_ptr()
        a.x, a.weight, a.y = rows.data_ptr(), weight.data_ptr(), y.data_ptr()
        with _lib.device_guard(dev):
            _lib.check(_lib.load().rwk_layer_norm_forward(ctypes.addressof(a), _lib.current_stream(dev)),
                       "rwk_layer_norm_forward")
    return y, rows, weight, stats, a


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, rows, weight, stats, ctx.args = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(rows, weight, stats)
        ctx.has_bias = bias is not None
        ctx.blocks = _lib.load().rwk_layer_norm_backward_blocks(stats.shape[1], x.shape[-1], ctx.args.type)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        # little is done here: the engine's thread has just woken up, and everything in it takes twice its time
        _lib.refuse_tangent(dy)
        rows, weight, stats = ctx.saved_tensors
        a, dev = _Args.from_buffer_copy(ctx.args), dy.device          # a copy: a graph may be walked by two threads
        rows, a.x_stride = _rows(rows)                    # hooks of saved tensors may have laid them anew
        weight, stats = weight.contiguous(), stats.contiguous()
        dx = torch.empty_like(dy, memory_format=torch.contiguous_format)
        dw, db = torch.empty((2, a.width), dtype=weight.dtype, device=dev).unbind(0)
        if a.rows == 0:
            dw.zero_()
            db.zero_()
        else:
            dy, a.dy_stride = _rows(dy)
            partials = torch.empty((ctx.blocks, 2 * a.width), dtype=torch.float32, device=dev)
            a.x, a.weight, a.mean, a.dy = rows.data_ptr(), weight.data_ptr(), stats.data_ptr(), dy.data_ptr()
            a.rstd = a.mean + 4 * a.rows
            a.dx, a.partials, a.dw, a.db = dx.data_ptr(), partials.data_ptr(), dw.data_ptr(), db.data_ptr()
            with _lib.device_guard(dev):
                _lib.check(_lib.load().rwk_layer_norm_backward(ctypes.addressof(a), _lib.current_stream(dev)),
                           "rwk_layer_norm_backward")
        return dx, dw, db if ctx.has_bias else None, None

def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor = None, eps: float = 1e-5) -> torch.Tensor:
    """``x`` (..., D) float32, float16 or bfloat16; ``weight`` and ``bias`` (D,) of the same type or both float32.
    Returns a contiguous tensor like ``x``.  Rows may lie any distance apart (a slice of a wider matrix is read in
    place).  Differentiable once with respect to all three."""
    _check(x, weight, bias)
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and
                                                                               bias.requires_grad)) or _lib.forward_mode():
        return _LayerNorm.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]


class LayerNorm(nn.Module):
    """:func:`layer_norm` with parameters ``weight`` (ones) and ``bias`` (zeros) of ``width`` elements."""

    def __init__(self, width: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None):
        super().__init__()
        self.eps = float(eps)
        self.weight = nn.Parameter(torch.ones(width, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(width, device=device, dtype=dtype)) if bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)
