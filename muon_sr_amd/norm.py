"""Layer norm and its gradients, the weight's and bias's among them.

    y = layer_norm(x, weight, bias)              # over the last dimension

Statistics and sums are formed in fp32, in an order that depends on the sizes alone: the same call gives
the same bits.  The reference's models (examples.py:56-82) use ``nn.LayerNorm``, whose place ``LayerNorm`` takes.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .experts import _ELEM, _elem, _once, _one_gpu
from .head import _flat_rows

__all__ = ["layer_norm", "LayerNorm"]


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        d = x.shape[-1]
        x2, ld = _flat_rows(x, d)
        rows = x2.shape[0]
        weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        mean, rstd = torch.empty((2, rows), dtype=torch.float32, device=x.device)
        vector = weight if weight is not None else bias
        welem = _ELEM[vector.dtype] if vector is not None else _lib.F32
        _lib.call(x, "msr_layer_norm", x2.data_ptr(), ld, _lib.ptr(weight), _lib.ptr(bias), eps, rows, d, y.data_ptr(),
                  mean.data_ptr(), rstd.data_ptr(), _ELEM[x.dtype], welem)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.welem, ctx.vector = welem, vector.dtype if vector is not None else None
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors     # saved-tensor hooks may have changed their strides
        d = x.shape[-1]
        (x2, ldx), (dy2, lddy) = _flat_rows(x, d), _flat_rows(dy, d)
        weight, mean, rstd = None if weight is None else weight.contiguous(), mean.contiguous(), rstd.contiguous()
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_x else None
        dw = torch.empty(d, dtype=ctx.vector, device=x.device) if want_w else None
        db = torch.empty(d, dtype=ctx.vector, device=x.device) if want_b else None
        size, ws = ctypes.c_size_t(), None
        if want_w or want_b:
            _lib.check(_lib.lib().msr_layer_norm_workspace_bytes(x2.shape[0], d, _ELEM[x.dtype], ctypes.byref(size)),
                       "msr_layer_norm_workspace_bytes")
            ws = _lib.workspace(x, size.value)
        _lib.call(x, "msr_layer_norm_grad", dy2.data_ptr(), lddy, x2.data_ptr(), ldx, _lib.ptr(weight), mean.data_ptr(), rstd.data_ptr(),
                  x2.shape[0], d, _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), _ELEM[x.dtype], ctx.welem, _lib.ptr(ws), size.value)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x`` (bf16 or fp32 [..., d]), in
    fp32, rounded once to x's type.  ``weight``, ``bias``: [d], both bf16 or both fp32, either may be left out; their gradients
    have their type."""
    given = [t for t in (weight, bias) if t is not None]
    _one_gpu("layer_norm", x, *given)
    _elem(x, "layer_norm: x")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm needs rows with elements, got {tuple(x.shape)}")
    for t in given:
        _elem(t, "layer_norm: weight and bias")
        if t.shape != x.shape[-1:] or t.dtype != given[0].dtype:
            raise ValueError(f"layer_norm needs a weight and bias of {x.shape[-1]} elements of one type")
    return _LayerNorm.apply(x, weight, bias, float(eps))


class LayerNorm(torch.nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension, computed by ``layer_norm``."""

    def __init__(self, normalized_shape, *args, **kwargs):
        super().__init__(normalized_shape, *args, **kwargs)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm normalizes the last dimension, got a shape of {len(self.normalized_shape)}")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() < 1 or x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"LayerNorm needs [..., {self.normalized_shape[0]}], got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
