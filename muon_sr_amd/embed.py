"""Embedding with scaling, and its gradient by sorted tokens.

    y = embedding(ids, weight, scale=scale)      # scale * weight[ids]

``SREmbedding`` is to ``nn.Embedding`` what ``SRLinear`` is to ``nn.Linear``: its gradient is added to
``weight.acc_grad`` with stochastic rounding, with the arithmetic, seeds and noise of ``TritonSRAccumulator``'s hook
(muon_sr/triton_adamw.py:206-229, 252-265), row by row of the words that the tokens hit, where the hook
reads a whole gradient and accumulator.  Sums are formed in fp32 in a fixed order: the same call gives the
same bits.  The reference's training loops call torch's embedding.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .experts import _one_gpu

__all__ = ["embedding", "embedding_grad_sr_accum", "SREmbedding"]


def embedding(ids: torch.Tensor, weight: torch.Tensor, padding_idx: int = None, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[ids]``, rounded once, as [*ids.shape, d].  ``weight``: bf16 or fp32 [vocab, d]; ``ids``: int32 or int64; one
    outside [0, vocab) has no word: its row is 0 and gives no gradient.  ``padding_idx`` gives none either (its row is
    looked up as any other).  The gradient goes to autograd, whole; ``SREmbedding`` adds it to its accumulator."""
    return _lib.nodes().embedding(ids, weight, padding_idx, scale, False)


def embedding_grad_sr_accum(weight: torch.Tensor, ids: torch.Tensor, dy: torch.Tensor, padding_idx: int = None,
                            scale: float = 1.0, seed: int = None) -> None:
    """``weight.acc_grad[v] <- SR(weight.acc_grad[v] + bf16(scale * sum of dy's rows of word v))`` for the words of ``ids``; the
    other rows are not touched.  ``weight``: bf16 [vocab, d], ``dy``: bf16 [*ids.shape, d].  The buffer is created (as
    zeros) on the first call, and one that is there has to be like it (ValueError); ``seed``: 32 bits, drawn from ``random``
    if not given, as the accumulator's hook draws it."""
    padding = _lib.nodes().check_embedding("embedding_grad_sr_accum", ids, weight, padding_idx)
    _one_gpu("embedding_grad_sr_accum", weight, dy)
    if weight.dtype != torch.bfloat16 or dy.dtype != torch.bfloat16:
        raise ValueError(f"embedding_grad_sr_accum needs bf16 tensors, got {weight.dtype} and {dy.dtype}")
    if dy.shape != (*ids.shape, weight.shape[1]):
        raise ValueError(f"embedding_grad_sr_accum needs dy of shape {(*ids.shape, weight.shape[1])}, got {tuple(dy.shape)}")
    vocab, d = weight.shape
    acc, drawn, first, noise = _lib.accumulator(weight, "embedding_grad_sr_accum", seed)
    ids, dy = ids.contiguous(), dy.reshape(ids.numel(), d)
    if len(dy) <= 1 or (d > 1 and dy.stride(1) != 1) or dy.stride(0) < d:
        dy = dy.contiguous()
    size = ctypes.c_size_t()
    _lib.check(_lib.lib().msr_embedding_workspace_bytes(len(dy), vocab, d, ctypes.byref(size)), "msr_embedding_workspace_bytes")
    ws = _lib.workspace(dy, size.value)
    _lib.call(weight, "msr_embedding_grad_sr_accum", ids.data_ptr(), int(ids.dtype == torch.int64), len(dy), dy.data_ptr(),
              max(d, dy.stride(0)), vocab, d, float(scale), padding, acc.data_ptr(), drawn, int(first), noise, None, _lib.ptr(ws), size.value)
    if first:
        weight.acc_grad = acc


class SREmbedding(torch.nn.Embedding):
    """``nn.Embedding`` (its rows scaled by ``scale``) whose gradient is added to ``weight.acc_grad`` with stochastic
    rounding (for training with ``TritonSRAccumulator``: ``reassign_grad_buffer`` then moves ``acc_grad`` to
    ``grad`` as for every other parameter).  The accumulator is the parameter's under activation checkpointing and other
    saved-tensor hooks too; the gradient of a parametrized weight, or of one that is not bf16, goes to autograd."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: int = None, scale: float = 1.0, device=None,
                 dtype=torch.bfloat16):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device, dtype=dtype)
        self.scale = float(scale)

    @classmethod
    def from_pretrained(cls, embeddings: torch.Tensor, freeze: bool = True, padding_idx: int = None, *, scale: float = 1.0):
        """The module whose weight is ``embeddings`` [vocab, d] (not a copy), frozen unless ``freeze`` is False; ``nn.Embedding``'s other options
        are not taken."""
        if embeddings.dim() != 2:
            raise ValueError(f"SREmbedding.from_pretrained needs embeddings [vocab, d], got {tuple(embeddings.shape)}")
        module = cls(*embeddings.shape, padding_idx=padding_idx, scale=scale, device="meta", dtype=embeddings.dtype)
        module.weight = torch.nn.Parameter(embeddings, requires_grad=not freeze)
        return module

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        weight = self.weight
        # a weight that is computed (a parametrization) holds nothing that lasts, and one that is not bf16 has no accumulator: autograd
        # gets the gradient
        accumulate = weight.is_leaf and weight.dtype == torch.bfloat16 and weight.requires_grad and torch.is_grad_enabled()
        return _lib.nodes().embedding(ids, weight, self.padding_idx, self.scale, accumulate)

    def extra_repr(self):
        return super().extra_repr() + (f", scale={self.scale}" if self.scale != 1.0 else "")
