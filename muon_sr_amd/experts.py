"""Mixture-of-experts layers: tokens sorted by expert and back, and the experts' products.

    order = order_tokens(ids, num_experts)          # ids [tokens, k] from the router's top-k
    rows = dispatch_tokens(x, order)                # a row per (token, choice), expert by expert
    rows = down(act(up(rows, order.offsets)), order.offsets)   # SRExperts: a linear layer per expert
    y = combine_tokens(rows, weights, order)        # the weighted sum of a token's rows

Nothing here waits for the GPU: how many rows each expert has is known there only
(``order.offsets``).  ``dispatch_tokens``, ``combine_tokens`` and ``expert_linear`` are
differentiable.  ``SRExperts`` is to ``expert_linear`` what ``SRLinear`` is to ``nn.Linear``:
its weight gradients are accumulated into ``weight.acc_grad`` with stochastic rounding inside
the weight-gradient product, with the arithmetic, seeds and noise of ``TritonSRAccumulator``'s hook
(muon_sr/triton_adamw.py:206-229, 252-265).  The reference has no mixture-of-experts code.
"""
from __future__ import annotations

import ctypes
import math
import random
from typing import NamedTuple

import torch

from . import _lib

__all__ = ["TokenOrder", "order_tokens", "dispatch_tokens", "combine_tokens", "expert_linear",
           "experts_wgrad_sr_accum", "SRExperts"]

MAX_ROW_STRIDE = 1 << 21   # of the experts' products
_ELEM = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


class TokenOrder(NamedTuple):
    """The rows of the slots (t, j), sorted by expert, earlier slots first.

    offsets   int32 [experts + 1]: expert e has the rows offsets[e] to offsets[e + 1] - 1
    position  int32 [tokens, k]: the row of a slot, -1 where it has no expert
    source    int32 [tokens * k]: the slot t * k + j of a row, -1 for the rows from offsets[-1] on
    """
    offsets: torch.Tensor
    position: torch.Tensor
    source: torch.Tensor


def _elem(t: torch.Tensor, what: str) -> int:
    code = _ELEM.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be bf16 or fp32, got {t.dtype}")
    return code


def _one_gpu(what: str, first: torch.Tensor, *others):
    device = first.get_device()
    if device < 0:
        _lib.require_gpu(first, what)
    for t in others:
        if t.get_device() != device:
            _lib.require_gpu(t, what)
            raise ValueError(f"{what} needs every tensor on one GPU")


def _once(backward):
    """``once_differentiable`` where a graph of the backward pass is made (a second derivative raises); else
    ``backward`` itself, which saves 12 us of host time per call."""
    guarded = torch.autograd.function.once_differentiable(backward)
    return lambda ctx, *grads: guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)


def order_tokens(ids: torch.Tensor, num_experts: int) -> TokenOrder:
    """Sorts the slots of ``ids`` (int32 or int64 [tokens, k]: the experts of each token) by expert.  A slot
    whose id is outside [0, num_experts) has no expert: it is dropped."""
    _one_gpu("order_tokens", ids)
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"order_tokens needs int32 or int64 ids, got {ids.dtype}")
    if ids.dim() != 2 or ids.shape[1] < 1:
        raise ValueError(f"order_tokens needs ids of shape [tokens, k], got {tuple(ids.shape)}")
    ids = ids.contiguous()
    tokens, k = ids.shape
    L, size = _lib.lib(), ctypes.c_size_t()
    _lib.check(L.msr_order_workspace_bytes(tokens, k, num_experts, ctypes.byref(size)), "msr_order_workspace_bytes")
    made = lambda *shape: torch.empty(shape, dtype=torch.int32, device=ids.device)  # noqa: E731
    order = TokenOrder(made(num_experts + 1), made(tokens, k), made(tokens * k))
    ws = made(size.value // 4) if size.value else None
    _lib.check(L.msr_order_tokens(ids.data_ptr(), int(ids.dtype == torch.int64), tokens, k, num_experts,
                                  order.offsets.data_ptr(), order.position.data_ptr(), order.source.data_ptr(),
                                  ws.data_ptr() if ws is not None else None, size.value, _lib.stream_of(ids)),
               "msr_order_tokens")
    return order


def _check_order(what: str, order: TokenOrder):
    offsets, position, source = order
    if not (offsets.dtype == position.dtype == source.dtype == torch.int32 and position.dim() == 2 and
            offsets.is_contiguous() and position.is_contiguous() and source.numel() == position.numel()):
        raise ValueError(f"{what}: order is not what order_tokens returned")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [n, d] with unit column stride, a row stride that the library takes and, where 16 bytes divide a row,
    16-byte aligned rows: a copy where it has none (one pass over t, where unaligned kernels would take as
    long for each of a token's rows)."""
    es, d, ld = t.element_size(), t.shape[1], t.stride(0)
    if t.stride(1) != 1 or ld < d or ld > MAX_ROW_STRIDE or (d * es % 16 == 0 and (ld * es % 16 or t.data_ptr() % 16)):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _contiguous(t: torch.Tensor) -> torch.Tensor:
    return _rows(t.contiguous())


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        tokens, k = order.position.shape
        d = x.shape[1]
        x = _rows(x)
        rows = torch.empty((tokens * k, d), dtype=x.dtype, device=x.device)
        _lib.check(_lib.lib().msr_dispatch(x.data_ptr(), x.stride(0), rows.data_ptr(), order.position.data_ptr(),
                                           order.offsets.data_ptr(), order.offsets.numel() - 1, tokens, k, d,
                                           _ELEM[x.dtype], _lib.stream_of(x)), "msr_dispatch")
        ctx.order = order
        return rows

    @staticmethod
    @_once
    def backward(ctx, drows):
        tokens, k = ctx.order.position.shape
        drows = _contiguous(drows)
        dx = torch.empty((tokens, drows.shape[1]), dtype=drows.dtype, device=drows.device)
        _lib.check(_lib.lib().msr_dispatch_grad(drows.data_ptr(), dx.data_ptr(), ctx.order.position.data_ptr(), tokens, k,
                                                drows.shape[1], _ELEM[drows.dtype], _lib.stream_of(drows)),
                   "msr_dispatch_grad")
        return dx, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order):
        tokens, k = order.position.shape
        rows, weights = _contiguous(rows), weights.contiguous()
        y = torch.empty((tokens, rows.shape[1]), dtype=rows.dtype, device=rows.device)
        _lib.check(_lib.lib().msr_combine(rows.data_ptr(), weights.data_ptr(), y.data_ptr(), order.position.data_ptr(),
                                          tokens, k, rows.shape[1], _ELEM[rows.dtype], _ELEM[weights.dtype],
                                          _lib.stream_of(rows)), "msr_combine")
        ctx.save_for_backward(rows, weights)
        ctx.order = order
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        rows, weights = ctx.saved_tensors     # saved-tensor hooks may have changed their strides
        rows, weights = _contiguous(rows), weights.contiguous()
        order = ctx.order
        tokens, k = order.position.shape
        d = rows.shape[1]
        dy = _rows(dy)
        drows = torch.empty_like(rows) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(weights) if ctx.needs_input_grad[1] else None
        _lib.check(_lib.lib().msr_combine_grad(dy.data_ptr(), dy.stride(0), rows.data_ptr(), weights.data_ptr(),
                                               drows.data_ptr() if drows is not None else None,
                                               dw.data_ptr() if dw is not None else None, order.position.data_ptr(),
                                               order.offsets.data_ptr(), order.offsets.numel() - 1, tokens, k, d,
                                               _ELEM[rows.dtype], _ELEM[weights.dtype], _lib.stream_of(rows)),
                   "msr_combine_grad")
        return drows, dw, None


def dispatch_tokens(x: torch.Tensor, order: TokenOrder) -> torch.Tensor:
    """Rows [tokens * k, d] of ``x`` (bf16 or fp32 [tokens, d]) in the order of ``order``; rows without a
    slot are 0.  A token's gradient is the sum over its rows, formed in fp32."""
    _one_gpu("dispatch_tokens", x, *order)
    _check_order("dispatch_tokens", order)
    _elem(x, "dispatch_tokens: x")
    if x.dim() != 2 or x.shape[0] != order.position.shape[0]:
        raise ValueError(f"dispatch_tokens needs x of shape [{order.position.shape[0]}, d], got {tuple(x.shape)}")
    return _Dispatch.apply(x, order)


def combine_tokens(rows: torch.Tensor, weights: torch.Tensor, order: TokenOrder) -> torch.Tensor:
    """y[t] = sum_j weights[t, j] * rows[order.position[t, j]] over the slots that have an expert, as
    [tokens, d]: sums in fp32, rounded once to the type of ``rows`` (bf16 or fp32).  ``weights``: bf16 or
    fp32 [tokens, k]; its gradient has its type."""
    _one_gpu("combine_tokens", rows, weights, *order)
    _check_order("combine_tokens", order)
    _elem(rows, "combine_tokens: rows")
    _elem(weights, "combine_tokens: weights")
    n = order.position.numel()
    if rows.dim() != 2 or rows.shape[0] != n or weights.shape != order.position.shape:
        raise ValueError(f"combine_tokens needs rows of shape [{n}, d] and weights of {tuple(order.position.shape)}, got "
                         f"{tuple(rows.shape)} and {tuple(weights.shape)}")
    return _Combine.apply(rows, weights, order)


# ---------------------------------------------------------------------------
# the experts' products
# ---------------------------------------------------------------------------

def _check_products(what, weight, offsets, x, dy=None):
    if weight.dim() != 3 or not weight.is_contiguous():
        raise ValueError(f"{what} needs a contiguous weight [experts, out, in], got {tuple(weight.shape)}")
    sides = [(x, weight.shape[2])] + ([(dy, weight.shape[1])] if dy is not None else [])
    _one_gpu(what, weight, offsets, *(t for t, _ in sides))
    if offsets.dtype != torch.int32 or offsets.shape != (weight.shape[0] + 1,) or not offsets.is_contiguous():
        raise ValueError(f"{what} needs int32 offsets of {weight.shape[0] + 1} entries (order_tokens gives them)")
    if any(t.dtype != torch.bfloat16 for t in (weight, *(t for t, _ in sides))):
        raise ValueError(f"{what} needs bf16 tensors")
    if weight.shape[1] % 8 or weight.shape[2] % 8:
        raise ValueError(f"{what} needs features that are multiples of 8, got {weight.shape[1]} x {weight.shape[2]}")
    for t, width in sides:
        if t.dim() != 2 or t.shape[1] != width or t.shape[0] != sides[0][0].shape[0]:
            raise ValueError(f"{what}: rows of shape {tuple(t.shape)} do not fit the weight {tuple(weight.shape)}")


def _forward(x, weight, offsets):
    E, o, i = weight.shape
    y = torch.empty((x.shape[0], o), dtype=torch.bfloat16, device=x.device)
    _lib.check(_lib.lib().msr_experts_forward(x.data_ptr(), x.stride(0), weight.data_ptr(), y.data_ptr(), offsets.data_ptr(),
                                              x.shape[0], E, i, o, _lib.stream_of(x)), "msr_experts_forward")
    return y


def _dgrad(dy, weight, offsets):
    E, o, i = weight.shape
    dx = torch.empty((dy.shape[0], i), dtype=torch.bfloat16, device=dy.device)
    _lib.check(_lib.lib().msr_experts_dgrad(dy.data_ptr(), dy.stride(0), weight.data_ptr(), dx.data_ptr(),
                                            offsets.data_ptr(), dy.shape[0], E, i, o, _lib.stream_of(dy)),
               "msr_experts_dgrad")
    return dx


def _wgrad(weight, x, dy, offsets):
    E, o, i = weight.shape
    dw = torch.empty_like(weight)
    _lib.check(_lib.lib().msr_experts_wgrad(dw.data_ptr(), x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0),
                                            offsets.data_ptr(), x.shape[0], E, i, o, _lib.stream_of(x)),
               "msr_experts_wgrad")
    return dw


def experts_wgrad_sr_accum(weight: torch.Tensor, x: torch.Tensor, dy: torch.Tensor, offsets: torch.Tensor,
                           seed: int = None) -> None:
    """``weight.acc_grad[e] <- SR(weight.acc_grad[e] + bf16(dy_e^T x_e))`` for every expert in one kernel: the
    counterpart of ``linear_wgrad_sr_accum`` for ``weight`` [experts, out, in] and rows sorted by expert.
    ``x``: bf16 [rows, in], ``dy``: bf16 [rows, out].  The buffer is created (as zeros) on the first
    call, and one that is there has to be like it (ValueError); ``seed``: 32 bits, drawn from ``random`` if not given, as the accumulator's hook draws it."""
    _check_products("experts_wgrad_sr_accum", weight, offsets, x, dy)
    x, dy = _rows(x), _rows(dy)
    first = not hasattr(weight, "acc_grad")
    if not first:
        _lib.check_accumulator(weight, "experts_wgrad_sr_accum")
    if seed is None:
        seed = random.getrandbits(32)
    acc = torch.empty_like(weight, memory_format=torch.contiguous_format) if first else weight.acc_grad
    E, o, i = weight.shape
    rc = _lib.lib().msr_experts_wgrad_sr_accum(acc.data_ptr(), x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0),
                                               offsets.data_ptr(), x.shape[0], E, i, o, seed, int(first),
                                               _lib.noise_mode(), None, _lib.stream_of(acc))
    _lib.check(rc, "msr_experts_wgrad_sr_accum")
    if first:
        weight.acc_grad = acc


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, accumulate):
        x = _rows(x)
        ctx.save_for_backward(x, weight, offsets)
        # the tensor that holds acc_grad: saved-tensor hooks (activation checkpointing, offloading) unpack another one.  A
        # weight that is computed (a parametrization) holds nothing that lasts, so its gradient goes to autograd.
        ctx.owner = weight if accumulate and weight.is_leaf else None
        return _forward(x, weight, offsets)

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, offsets = ctx.saved_tensors     # saved-tensor hooks may have changed their strides
        x, weight, offsets, dy = _rows(x), weight.contiguous(), offsets.contiguous(), _rows(dy)
        dx = _dgrad(dy, weight, offsets) if ctx.needs_input_grad[0] else None
        dw = None
        if ctx.needs_input_grad[1]:
            if ctx.owner is not None:
                experts_wgrad_sr_accum(ctx.owner, x, dy, offsets)
            else:
                dw = _wgrad(weight, x, dy, offsets)
        return dx, dw, None, None


def expert_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """y[r] = weight[e] @ x[r] for the rows r of each expert e (``offsets[e]`` to ``offsets[e + 1] - 1``), bf16
    with fp32 accumulation.  ``x``: [rows, in], ``weight``: [experts, out, in], in and out multiples of
    8.  Rows from ``offsets[-1]`` on give 0 and get a zero gradient.  The weight gradient goes to autograd
    (``TritonSRAccumulator``'s hook accumulates it as any other); ``SRExperts`` accumulates it in the product."""
    _check_products("expert_linear", weight, offsets, x)
    return _ExpertLinear.apply(x, weight, offsets, False)


class SRExperts(torch.nn.Module):
    """A linear layer without bias for each expert, for rows sorted by expert, whose weight gradients are
    accumulated into ``weight.acc_grad`` with stochastic rounding inside the weight-gradient product (for
    training with ``TritonSRAccumulator``: ``reassign_grad_buffer`` then moves ``acc_grad`` to ``grad``
    as for every other parameter).  ``weight`` is [experts, out, in], initialised as ``nn.Linear``'s; the
    Muon classes orthogonalise each expert's matrix by itself.  The accumulator is the parameter's under activation
    checkpointing and other saved-tensor hooks too; a parametrized weight's gradient goes to autograd."""

    def __init__(self, num_experts: int, in_features: int, out_features: int, device=None, dtype=torch.bfloat16):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.empty((num_experts, out_features, in_features), device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self):
        bound = 1.0 / math.sqrt(self.weight.shape[2])
        torch.nn.init.uniform_(self.weight, -bound, bound)

    def forward(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        _check_products("SRExperts", self.weight, offsets, x)
        return _ExpertLinear.apply(x, self.weight, offsets, True)

    def extra_repr(self):
        E, o, i = self.weight.shape
        return f"num_experts={E}, in_features={i}, out_features={o}"
