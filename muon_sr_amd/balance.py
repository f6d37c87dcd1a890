"""A mixture-of-experts router's balance loss and the slots per expert.

    loss, counts = balance_loss(logits, ids)     # logits [tokens, experts], ids [tokens, k] of the router's top-k

loss = experts * sum_e (share of the slots with e) * (mean over tokens of softmax(logits)[e]); 1 where
both are even.  The probabilities are never in memory.  Stands beside ``order_tokens``, whose ids it takes.
The reference has no mixture-of-experts code.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .experts import _ELEM, _elem, _once, _one_gpu
from .head import _flat_rows

__all__ = ["balance_loss"]


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask):
        tokens, experts = logits.shape
        rows, ld = _flat_rows(logits, experts)
        ids = ids.contiguous()
        mask = None if mask is None else mask.contiguous()
        f32 = dict(dtype=torch.float32, device=logits.device)
        loss, lse, slope = torch.empty((), **f32), torch.empty(tokens, **f32), torch.empty(experts, **f32)
        counts = torch.empty(experts, dtype=torch.int32, device=logits.device)
        size = ctypes.c_size_t()
        _lib.check(_lib.lib().msr_balance_workspace_bytes(tokens, experts, ctypes.byref(size)), "msr_balance_workspace_bytes")
        ws = _lib.workspace(logits, size.value)
        _lib.call(logits, "msr_balance_loss", rows.data_ptr(), ld, ids.data_ptr(), int(ids.dtype == torch.int64), _lib.ptr(mask), tokens,
                  experts, ids.shape[1], loss.data_ptr(), counts.data_ptr(), lse.data_ptr(), slope.data_ptr(), _ELEM[logits.dtype],
                  ws.data_ptr(), size.value)
        ctx.save_for_backward(logits, mask, lse, slope)
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    @_once
    def backward(ctx, dloss, _):
        logits, mask, lse, slope = ctx.saved_tensors     # saved-tensor hooks may have changed their strides
        tokens, experts = logits.shape
        rows, ld = _flat_rows(logits, experts)
        mask, lse, slope = None if mask is None else mask.contiguous(), lse.contiguous(), slope.contiguous()
        out = torch.empty((tokens, experts), dtype=logits.dtype, device=logits.device)
        _lib.call(logits, "msr_balance_grad", rows.data_ptr(), ld, _lib.ptr(mask), lse.data_ptr(), slope.data_ptr(),
                  dloss.data_ptr(), tokens, experts, out.data_ptr(), _ELEM[logits.dtype])
        return out, None, None


def balance_loss(logits: torch.Tensor, ids: torch.Tensor, mask: torch.Tensor = None):
    """The balance loss (fp32, differentiable in ``logits``) and the number of slots of each expert (int32 [experts]).  ``logits``:
    bf16 or fp32 [tokens, experts]; ``ids``: int32 or int64 [tokens, k], the experts chosen for each token, slots outside [0,
    experts) being dropped; ``mask``: bool [tokens], the tokens that count (padding does not: its logits reach nothing).  The loss is
    0 where none does.  Logits of -inf have probability 0."""
    _one_gpu("balance_loss", logits, ids, *([] if mask is None else [mask]))
    _elem(logits, "balance_loss: logits")
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"balance_loss needs int32 or int64 ids, got {ids.dtype}")
    if logits.dim() != 2 or ids.dim() != 2 or ids.shape[0] != logits.shape[0] or ids.shape[1] < 1 or \
            not 1 <= logits.shape[1] <= _lib.EXPERTS_MAX:
        raise ValueError(f"balance_loss needs logits [tokens, experts] with 1 to {_lib.EXPERTS_MAX} experts and ids [tokens, k], got "
                         f"{tuple(logits.shape)} and {tuple(ids.shape)}")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != logits.shape[:1]):
        raise ValueError(f"balance_loss needs a bool mask of {logits.shape[0]} tokens, got {mask.dtype} {tuple(mask.shape)}")
    return _Balance.apply(logits, ids, mask)
