"""The global norm of many gradients and clipping by it, between backward and ``step()``.

    loss.backward()
    TritonSRAccumulator.reassign_grad_buffer(model)
    norm = clip_grad_norm_(model.parameters(), 1.0)
    opt.step()

``clip_grad_norm_`` takes the place of ``torch.nn.utils.clip_grad_norm_`` (the reference's
training loops would call that one): the same arguments and treatment of non-finite norms, for
bf16 and fp32 gradients on one GPU and the norms 1, 2 and inf (others are refused); many tensors
per kernel launch, sums in 64 bits, and a norm in fp32 whatever the gradients' type.  Nothing
synchronises with the host, except for ``error_if_nonfinite``.
"""
from __future__ import annotations

import ctypes
import math
import operator
import struct
from array import array

import torch

from . import _lib

__all__ = ["grad_norm", "clip_grads", "clip_grad_norm_"]

_NORMS = {1.0: _lib.NORM_1, 2.0: _lib.NORM_2, math.inf: _lib.NORM_INF}
_pack_item = struct.Struct("=QQqii").pack   # msr_clip_item
_T, _dtype = torch.Tensor, operator.attrgetter("dtype")


def _norm_code(norm_type) -> int:
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 1, 2 or inf (got {norm_type!r})")
    return code


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill its memory without gaps or overlaps, in some order of its dims."""
    if t.is_contiguous():
        return True
    order = sorted(range(t.dim()), key=lambda i: (t.stride(i), t.shape[i]), reverse=True)
    return t.permute(order).is_contiguous()


def _check(t: torch.Tensor, device, what: str):
    if t.layout is not torch.strided:
        raise RuntimeError(f"{what} does not support sparse gradients")
    if t.dtype != torch.bfloat16 and t.dtype != torch.float32:
        raise ValueError(f"{what} supports bf16 or fp32 gradients, got {t.dtype}")
    if not t.is_cuda:
        _lib.require_gpu(t, what)
    if t.get_device() != device:
        raise ValueError(f"{what} needs every gradient on one GPU")


def _plain(tensors, device):
    """Contiguous bf16 tensors on that GPU."""
    return set(map(_T.get_device, tensors)) == {device} and set(map(_dtype, tensors)) == {torch.bfloat16} and \
        all(map(_T.is_contiguous, tensors))


def _items(grads, outs, device, what):
    """The list's msr_clip_items, what has to live until they are used, and the outs to copy results to."""
    # The common case by maps over the list: host time bounds many small tensors (73 gradients, out of place: 98 us
    # a call with the loop below, 52 so).
    if device >= 0 and _plain(grads, device) and (outs is None or outs is grads or (
            _plain(outs, device) and all(map(_T.is_same_size, grads, outs)))):
        a = array("q", bytes(32 * len(grads)))
        a[0::4] = array("q", map(_T.data_ptr, grads))
        if outs is not None:
            a[1::4] = a[0::4] if outs is grads else array("q", map(_T.data_ptr, outs))
        a[2::4] = array("q", map(_T.numel, grads))
        return a.tobytes(), (), ()
    with torch.no_grad():
        return _mixed_items(grads, outs, device, what)


def _mixed_items(grads, outs, device, what):
    f32 = torch.float32
    items, keep, back = [], [], []
    for i, g in enumerate(grads):
        o = None if outs is None else outs[i]
        _check(g, device, what)
        flags = _lib.CLIP_GRAD_F32 if g.dtype is f32 else 0
        src, dst = g, o
        if o is not None:
            _check(o, device, what)
            if o.shape != g.shape:
                raise ValueError(f"{what}: out {i} has shape {tuple(o.shape)}, its gradient {tuple(g.shape)}")
            if o.dtype is f32 and not flags:
                raise ValueError(f"{what}: out {i} is fp32, its gradient bf16")
            if o.dtype is f32:
                flags |= _lib.CLIP_OUT_F32
            # elements may be walked in memory order where both tensors have the same one
            if not (g.is_contiguous() and o.is_contiguous()) and not (g.stride() == o.stride() and _dense(g)):
                src = g.contiguous()
                dst = torch.empty(o.shape, dtype=o.dtype, device=o.device)
                back.append((o, dst))
        elif not _dense(g):
            src = g.contiguous()
        if src is not g:
            keep.append(src)
        items.append(_pack_item(src.data_ptr(), dst.data_ptr() if dst is not None else 0, src.numel(), flags, 0))
    return b"".join(items), keep, back


def _run(grads, outs, norm_type, max_norm, what):
    """The norm of ``grads`` and, with ``outs``, the clipped gradients written there."""
    code, device, n = _norm_code(norm_type), grads[0].get_device(), len(grads)
    items, keep, back = _items(grads, outs, device, what)
    norm = torch.empty((), dtype=torch.float32, device=torch.device("cuda", device))
    L, size = _lib.lib(), ctypes.c_size_t()
    _lib.check(L.msr_grad_norm_workspace_bytes(items, n, ctypes.byref(size)), "msr_grad_norm_workspace_bytes")
    ws = torch.empty(max(8, size.value), dtype=torch.uint8, device=norm.device)
    stream = _lib.stream_of(norm)
    if outs is None:
        _lib.check(L.msr_grad_norm(items, n, code, norm.data_ptr(), ws.data_ptr(), ws.numel(), stream), "msr_grad_norm")
    else:
        _lib.check(L.msr_clip_grads(items, n, code, max_norm, norm.data_ptr(), ws.data_ptr(), ws.numel(), stream),
                   "msr_clip_grads")
    if back:
        with torch.no_grad():
            for o, dst in back:
                o.copy_(dst)
    return norm


def grad_norm(grads, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of ``grads`` (a tensor, or an iterable of bf16 and fp32 tensors on one
    GPU; ``norm_type`` 1, 2 or inf) as a 0-dim fp32 tensor on that GPU; 0 for an empty list."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if not grads:
        return torch.tensor(0.0)
    return _run(grads, None, norm_type, 0.0, "grad_norm")


def clip_grads(grads, max_norm: float, norm_type: float = 2.0, out=None) -> torch.Tensor:
    """Scales ``grads`` by min(1, max_norm / (norm + 1e-6)), in place or, with ``out`` (a tensor for each
    gradient: of its type, or bf16 for an fp32 one, say the ``.grad`` that an optimizer of bf16
    parameters will read), into ``out``.  Returns the norm before clipping, as ``grad_norm`` does.
    The product is formed in fp32 and rounded once.  A NaN norm makes every gradient NaN, an infinite one
    makes the finite gradients 0, as in torch.  Tensors that share memory are refused, except that sharing is
    not noticed between tensors with gaps between their elements, which go through copies."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    outs = grads if out is None else [out] if isinstance(out, torch.Tensor) else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"clip_grads: {len(outs)} outs for {len(grads)} gradients")
    if not grads:
        return torch.tensor(0.0)
    return _run(grads, outs, norm_type, float(max_norm), "clip_grads")


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    foreach: bool = None) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` for bf16 and fp32 gradients on one GPU and norms 1, 2 and inf: clips
    the ``.grad`` of ``parameters`` in place and returns their norm (fp32).  With ``error_if_nonfinite`` the norm is
    waited for, and a non-finite one raises RuntimeError with the gradients as they were.  ``foreach``, which
    chooses an implementation in torch, changes nothing."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite:
        norm = grad_norm(grads, norm_type)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients from `parameters` is non-finite, "
                               "so it cannot be clipped. To disable this error and scale the gradients by the non-finite "
                               "norm anyway, set `error_if_nonfinite=False`")
    return clip_grads(grads, max_norm, norm_type)
