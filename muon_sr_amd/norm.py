"""Layer norm and its gradients, the weight's and bias's among them.

    y = layer_norm(x, weight, bias)              # over the last dimension

Statistics and sums are formed in fp32, in an order that depends on the sizes alone: the same call gives
the same bits.  The reference's models (examples.py:56-82) use ``nn.LayerNorm``, whose place ``LayerNorm`` takes.
"""
from __future__ import annotations

import torch

from . import _lib

__all__ = ["layer_norm", "LayerNorm"]


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x`` (bf16 or fp32 [..., d]), in
    fp32, rounded once to x's type.  ``weight``, ``bias``: [d], both bf16 or both fp32, either may be left out; their gradients
    have their type."""
    return _lib.nodes().layer_norm(x, weight, bias, eps)


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
