"""Layer norm over the last dimension: ``y = (x - mean) / sqrt(var + eps) * weight + bias`` per row, forward and
backward on the kernels of ``csrc/rwk_layer_norm.hip``.

The per-row companion of the head's batch norm (``rwgnn2/model.py:21,68``) for node features, walk steps and other
wide rows: float32, float16 or bfloat16 rows of any width, weights of the same type or float32.  All sums are fp32 in
a fixed order, with one rounding to the element type at the end, so results are bitwise reproducible.  HIP devices
only.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib

__all__ = ["layer_norm", "LayerNorm"]


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as (rows, width) with adjacent elements in a row and rows at least a width apart; a view if it can be."""
    t = t.reshape(-1, t.shape[-1])
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check(x, weight, bias):
    if not x.is_cuda:
        raise RuntimeError("gnn_amd runs on HIP devices only (no CPU fallback)")
    _lib.element_type(x.dtype)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("x needs a last dimension of at least one")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise ValueError(f"{name} has shape {tuple(t.shape)} for rows of {x.shape[-1]}")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise TypeError(f"{name} must have the type of x or float32")
        if t.device != x.device:
            raise RuntimeError(f"x and {name} must be on the same device")
    if bias is not None and bias.dtype != weight.dtype:
        raise TypeError("weight and bias must have the same type")


def _forward(x, weight, bias, eps, stats):
    """(y, mean, rstd, rows): ``rows`` is x as the kernel read it."""
    rows = _rows(x)
    n, width = rows.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty((2, n), dtype=torch.float32, device=x.device).unbind(0)
    if n:
        w = weight.contiguous()
        b = None if bias is None else bias.contiguous()
        with _lib.device_guard(x.device):
            _lib.check(_lib.load().rwk_layer_norm_forward(
                rows.data_ptr(), _stride(rows), w.data_ptr(), _lib.ptr(b), n, width, _lib.element_type(x.dtype),
                _lib.element_type(w.dtype), eps, y.data_ptr(), _lib.ptr(mean), _lib.ptr(rstd),
                _lib.current_stream(x.device)), "rwk_layer_norm_forward")
    return y, mean, rstd, rows


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd, rows = _forward(x.detach(), weight.detach(), None if bias is None else bias.detach(), eps, True)
        ctx.save_for_backward(rows, weight, mean, rstd)
        ctx.has_bias = bias is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        rows, weight, mean, rstd = ctx.saved_tensors
        n, width = rows.shape
        shape = dy.shape
        # one allocation for dw and db
        dwb = torch.empty((2, width), dtype=weight.dtype, device=rows.device)
        if n == 0:
            dwb.zero_()
            return torch.empty(shape, dtype=rows.dtype, device=rows.device), dwb[0], \
                dwb[1] if ctx.has_bias else None, None
        dy = _rows(dy)
        w = weight.contiguous()
        lib = _lib.load()
        code = _lib.element_type(rows.dtype)
        dx = torch.empty(shape, dtype=rows.dtype, device=rows.device)
        blocks = lib.rwk_layer_norm_backward_blocks(n, width, code)
        partials = torch.empty((blocks, 2 * width), dtype=torch.float32, device=rows.device)
        dw, db = dwb.unbind(0)
        with _lib.device_guard(rows.device):
            _lib.check(lib.rwk_layer_norm_backward(
                rows.data_ptr(), _stride(rows), dy.data_ptr(), _stride(dy), w.data_ptr(), mean.data_ptr(),
                rstd.data_ptr(), n, width, code, _lib.element_type(w.dtype), dx.data_ptr(), partials.data_ptr(),
                dw.data_ptr(), db.data_ptr(), _lib.current_stream(rows.device)), "rwk_layer_norm_backward")
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
                                                                               bias.requires_grad)):
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
