"""A language model's head with its softmax cross entropy, without the logits in memory.

    loss = linear_cross_entropy(x, weight, target)     # F.cross_entropy(F.linear(x, weight), target)

``SRHead`` is ``SRLinear`` for the head (its call gives logits) with a ``loss`` whose weight
gradient is accumulated into ``weight.acc_grad`` with stochastic rounding inside the product, with the arithmetic, seeds and
noise of ``TritonSRAccumulator``'s hook (muon_sr/triton_adamw.py:206-229, 252-265).  Logits exist
a tile at a time: the forward pass keeps each row's log-sum-exp, the backward pass forms them again, a piece of
the vocabulary at a time.  Rows of ``ignore_index`` cost nothing, and what they hold (NaN too) reaches neither the loss
nor a gradient.  The reference's training loops call torch's cross entropy on a linear layer.
"""
from __future__ import annotations

import ctypes
import random

import torch

from . import _lib
from .experts import _once
from .linear import SRLinear

__all__ = ["linear_cross_entropy", "SRHead"]


def _flat_rows(t: torch.Tensor, d: int):
    """t [..., d] as rows of unit column stride, and their stride."""
    t = t.reshape(t.shape[:-1].numel(), d)
    if t.shape[0] <= 1:
        return t.contiguous(), d
    if (t.stride(1) != 1 and d > 1) or t.stride(0) < d:
        t = t.contiguous()
    return t, t.stride(0)


def _packed(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _sizes(rows, vocab, d):
    forward, backward = ctypes.c_size_t(), ctypes.c_size_t()
    _lib.check(_lib.lib().msr_head_workspace_bytes(rows, vocab, d, ctypes.byref(forward), ctypes.byref(backward)),
               "msr_head_workspace_bytes")
    return forward.value, backward.value


class _Accumulating(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        vocab, d = weight.shape
        rows2, ld = _flat_rows(x, d)
        rows, target = rows2.shape[0], target.contiguous()
        packed = torch.empty((rows, d), dtype=torch.bfloat16, device=x.device)
        kept = torch.empty(3 * rows + 1, dtype=torch.int32, device=x.device)
        lse = torch.empty(rows, dtype=torch.float32, device=x.device)
        loss = torch.empty(target.shape if reduction == 0 else (), dtype=torch.float32, device=x.device)
        size, _ = _sizes(rows, vocab, d)
        ws = _lib.workspace(x, size)
        _lib.call(x, "msr_head_forward", rows2.data_ptr(), ld, weight.data_ptr(), target.data_ptr(), int(target.dtype == torch.int64),
                  ignore_index, rows, vocab, d, reduction, packed.data_ptr(), kept.data_ptr(), lse.data_ptr(), loss.data_ptr(),
                  _lib.ptr(ws), size)
        ctx.save_for_backward(packed, weight, kept, lse)
        ctx.shape, ctx.reduction = x.shape, reduction
        # the tensor that holds acc_grad: saved-tensor hooks (activation checkpointing, offloading) unpack another one
        ctx.owner = weight
        return loss

    @staticmethod
    @_once
    def backward(ctx, dloss):
        packed, weight, kept, lse = ctx.saved_tensors     # saved-tensor hooks may have changed their strides
        packed, weight, kept, lse = _packed(packed), _packed(weight), kept.contiguous(), lse.contiguous()
        vocab, d = weight.shape
        rows, dloss, owner = packed.shape[0], dloss.contiguous(), ctx.owner
        first = not hasattr(owner, "acc_grad")
        if not first:
            _lib.check_accumulator(owner, "SRHead")
        seed = random.getrandbits(32)
        acc = torch.empty_like(owner, memory_format=torch.contiguous_format) if first else owner.acc_grad
        dx = torch.empty(ctx.shape, dtype=torch.bfloat16, device=packed.device) if ctx.needs_input_grad[0] else None
        _, size = _sizes(rows, vocab, d)
        ws = _lib.workspace(packed, size)
        _lib.call(packed, "msr_head_backward", packed.data_ptr(), weight.data_ptr(), kept.data_ptr(), lse.data_ptr(), dloss.data_ptr(),
                  rows, vocab, d, ctx.reduction, _lib.ptr(dx), acc.data_ptr(), _lib.noise_mode(), seed, int(first), None, _lib.ptr(ws), size)
        if first:
            owner.acc_grad = acc
        return dx, None, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """The softmax cross entropy of the logits ``x @ weight.T`` with the words ``target``, fp32, differentiable.  ``x``: bf16
    [..., d], ``weight``: bf16 [vocab, d], d a multiple of 8; ``target``: int32 or int64 [...].  ``reduction``
    ``"none"`` gives a loss per row, 0 for ignored ones, ``"sum"`` and ``"mean"`` sum them, over the rows that are not
    ignored (0 where all are: torch's mean is NaN there).  Any other target outside [0, vocab) gives NaN, in the loss
    and the gradients.  The gradients are bf16, of products with fp32 accumulation; the weight gradient
    goes to autograd (``TritonSRAccumulator``'s hook accumulates it as any other)."""
    return _lib.nodes().linear_cross_entropy(x, weight, target, ignore_index, reduction)


class SRHead(SRLinear):
    """The head of a language model: ``SRLinear`` without bias (calling it gives logits), with ``loss(x, target)``,
    ``linear_cross_entropy`` whose weight gradient is accumulated into ``weight.acc_grad`` with stochastic rounding
    inside the product (for training with ``TritonSRAccumulator``).  The accumulator is the
    parameter's under activation checkpointing and other saved-tensor hooks too; a parametrized weight's
    gradient goes to autograd."""

    def __init__(self, in_features: int, vocab: int, device=None, dtype=torch.bfloat16):
        super().__init__(in_features, vocab, bias=False, device=device, dtype=dtype)

    def loss(self, x: torch.Tensor, target: torch.Tensor, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
        weight = self.weight
        # a weight that is computed (a parametrization) holds nothing that lasts: autograd gets its gradient
        if not (weight.is_leaf and weight.requires_grad and torch.is_grad_enabled()):
            return linear_cross_entropy(x, weight, target, ignore_index, reduction)
        code = _lib.nodes().check_head("SRHead", x, weight, target, reduction)
        return _Accumulating.apply(x, weight, target, ignore_index, code)
