"""A language model's head with its softmax cross entropy, without the logits in memory.

    loss = linear_cross_entropy(x, weight, target)     # F.cross_entropy(F.linear(x, weight), target)

``SRHead`` is ``SRLinear`` for the head (its call gives logits) with a ``loss`` whose weight
gradient is accumulated into ``weight.acc_grad`` with stochastic rounding inside the product, with the arithmetic, seeds and
noise of ``TritonSRAccumulator``'s hook (muon_sr/triton_adamw.py:206-229, 252-265).  Logits exist
a tile at a time: the forward pass keeps a number near each row's largest logit and the sum of its exponentials from there, the backward
pass forms the logits again, a piece of the vocabulary at a time.  Rows of ``ignore_index`` cost nothing, and what they hold (NaN too) reaches neither the
loss nor a gradient.  The reference's training loops call torch's cross entropy on a linear layer.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .linear import SRLinear

__all__ = ["linear_cross_entropy", "SRHead"]


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """The softmax cross entropy of the logits ``x @ weight.T`` with the words ``target``, fp32, differentiable.  ``x``: bf16
    [..., d], ``weight``: bf16 [vocab, d], d a multiple of 8; ``target``: int32 or int64 [...].  ``reduction``
    ``"none"`` gives a loss per row, 0 for ignored ones, ``"sum"`` and ``"mean"`` sum them, over the rows that are not
    ignored (0 where all are: torch's mean is NaN there).  Any other target outside [0, vocab) gives NaN, in the loss
    and the gradients.  The gradients are bf16, of products with fp32 accumulation whose operand, the logits' gradient, is bf16 too, as
    in a training loop in bf16; the weight gradient goes to autograd (``TritonSRAccumulator``'s hook accumulates it as any other)."""
    return _lib.nodes().linear_cross_entropy(x, weight, target, ignore_index, reduction, False)


class SRHead(SRLinear):
    """The head of a language model: ``SRLinear`` without bias (calling it gives logits), with ``loss(x, target)``,
    ``linear_cross_entropy`` whose weight gradient is accumulated into ``weight.acc_grad`` with stochastic rounding
    inside the product (for training with ``TritonSRAccumulator``).  The accumulator is the
    parameter's under activation checkpointing and other saved-tensor hooks too; a parametrized weight's
    gradient goes to autograd.

    ``loss`` is a call of the module: its forward hooks and pre-hooks run, with ``loss``'s arguments and its result (those of a
    subclass with a ``forward`` of its own, which takes ``x`` alone, do not)."""

    def __init__(self, in_features: int, vocab: int, device=None, dtype=torch.bfloat16):
        super().__init__(in_features, vocab, bias=False, device=device, dtype=dtype)

    def forward(self, x: torch.Tensor, *loss):
        """Logits; with the other arguments of ``loss``, the loss."""
        if not loss:
            return super().forward(x)
        weight = self.weight
        # a weight that is computed (a parametrization) holds nothing that lasts: autograd gets its gradient
        accumulate = weight.is_leaf and weight.requires_grad and torch.is_grad_enabled()
        return _lib.nodes().linear_cross_entropy(x, weight, *loss, accumulate)

    def loss(self, x: torch.Tensor, target: torch.Tensor, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
        # (a hook may compute the weight, as torch.nn.utils.weight_norm's does)
        call = self if getattr(type(self), "forward", None) is SRHead.forward else functools.partial(SRHead.forward, self)
        return call(x, target, ignore_index, reduction)
