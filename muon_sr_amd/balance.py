"""A mixture-of-experts router's balance loss and the slots per expert.

    loss, counts = balance_loss(logits, ids)     # logits [tokens, experts], ids [tokens, k] of the router's top-k

loss = experts * sum_e (share of the slots with e) * (mean over tokens of softmax(logits)[e]); 1 where
both are even.  The probabilities are never in memory.  Stands beside ``order_tokens``, whose ids it takes.
The reference has no mixture-of-experts code.
"""
from __future__ import annotations

import torch

from . import _lib

__all__ = ["balance_loss"]


def balance_loss(logits: torch.Tensor, ids: torch.Tensor, mask: torch.Tensor = None):
    """The balance loss (fp32, differentiable in ``logits``) and the number of slots of each expert (int32 [experts]).  ``logits``:
    bf16 or fp32 [tokens, experts]; ``ids``: int32 or int64 [tokens, k], the experts chosen for each token, slots outside [0,
    experts) being dropped; ``mask``: bool [tokens], the tokens that count (padding does not: its logits reach nothing).  The loss is
    0 where none does.  Logits of -inf have probability 0."""
    return _lib.nodes().balance_loss(logits, ids, mask)
