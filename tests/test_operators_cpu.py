"""Refusals of the gradient-norm, token and experts entry points that need no GPU (nothing is launched:
arguments are checked before any HIP call; addresses are made up)."""
import ctypes
import math

import pytest
import torch

ARG, ALIGN, WORKSPACE, OVERLAP = 1001, 1002, 1004, 1005
A, B, C, D, E, W = (i << 32 for i in range(1, 7))


@pytest.fixture(scope="module")
def lib():
    from muon_sr_amd import _lib
    return _lib.lib()


def items(*rows):
    from muon_sr_amd import _lib
    return (_lib.ClipItem * len(rows))(*[_lib.ClipItem(*r, 0) for r in rows]), len(rows)


def clip(lib, rows, norm=2, out=D, ws=W, ws_bytes=1 << 20):
    return lib.msr_clip_grads(*items(*rows), norm, 1.0, out, ws, ws_bytes, None)


def test_clip(lib):
    size = ctypes.c_size_t()
    assert lib.msr_grad_norm_workspace_bytes(*items((A, 0, 10 << 20, 0)), ctypes.byref(size)) == 0 and 8 <= size.value <= 1 << 16
    assert lib.msr_grad_norm_workspace_bytes(None, 0, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.msr_grad_norm_workspace_bytes(None, 1, ctypes.byref(size)) == ARG
    assert clip(lib, [(A, A, -1, 0)]) == ARG
    assert clip(lib, [(0, A, 5, 0)]) == ARG and clip(lib, [(A, 0, 5, 0)]) == ARG
    assert clip(lib, [(A, A, 5, 4)]) == ARG and clip(lib, [(A, B, 5, 2)]) == ARG      # unknown flag; bf16 into fp32
    assert clip(lib, [(A, A, 5, 0)], norm=7) == ARG and clip(lib, [(A, A, 5, 0)], out=None) == ARG
    assert clip(lib, [(A + 1, A + 1, 5, 0)]) == ALIGN and clip(lib, [(A + 2, B, 5, 1)]) == ALIGN
    assert clip(lib, [(A, A, 5, 0)], ws=W + 4) == ALIGN
    assert clip(lib, [(A, A, 5, 0)], ws_bytes=4) == WORKSPACE and b"workspace" in lib.msr_last_error()
    assert clip(lib, [(A, A + 2, 100, 0)]) == OVERLAP                                 # out inside its own grad
    assert clip(lib, [(A, A, 100, 1)]) == OVERLAP                                     # fp32 grad, bf16 out in its place
    assert clip(lib, [(A, A, 100, 0), (A + 100, B, 100, 0)]) == OVERLAP               # an out in another's grad
    assert clip(lib, [(A, C, 100, 0), (B, C + 100, 100, 0)]) == OVERLAP
    assert lib.msr_grad_norm(*items((A, 0, 100, 0)), 2, A + 40, W, 1 << 20, None) == OVERLAP
    assert clip(lib, [(A, B, 100, 0)], out=B + 8) == OVERLAP and clip(lib, [(A, W, 100, 0)]) == OVERLAP


def test_order(lib):
    size = ctypes.c_size_t()
    assert lib.msr_order_workspace_bytes(10, 2, 8, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.msr_order_workspace_bytes(100000, 8, 64, ctypes.byref(size)) == 0 and size.value > 0
    order = lambda *a, ws=W, n=1 << 30: lib.msr_order_tokens(*a, ws, n, None)  # noqa: E731
    for tokens, k, experts in ((-1, 2, 8), (10, 0, 8), (10, 2, 0), (10, 2, 1025), (1 << 30, 1, 8), (1 << 28, 4, 8)):
        assert order(A, 1, tokens, k, experts, B, C, D) == ARG
    assert order(None, 1, 10, 2, 8, B, C, D) == ARG and order(A, 1, 10, 2, 8, None, C, D) == ARG
    assert order(A + 4, 1, 10, 2, 8, B, C, D) == ALIGN and order(A, 0, 10, 2, 8, B + 2, C, D) == ALIGN
    assert order(A, 1, 100000, 8, 64, B, C, D, n=16) == WORKSPACE and order(A, 1, 100000, 8, 64, B, C, D, ws=None) == WORKSPACE
    assert order(A, 1, 10, 2, 8, B, C, C + 40) == OVERLAP and order(A, 1, 10, 2, 8, A, C, D) == OVERLAP


def test_passes(lib):
    disp = lambda x=A, ldx=16, rows=B, pos=C, off=D, E_=8, t=10, k=2, d=16, elem=0: lib.msr_dispatch(  # noqa: E731
        x, ldx, rows, pos, off, E_, t, k, d, elem, None)
    assert disp(t=0) == 0 and disp(d=0) == 0
    assert disp(x=None) == ARG and disp(ldx=15) == ARG and disp(elem=2) == ARG and disp(k=0) == ARG and disp(t=-1) == ARG
    assert disp(t=1 << 30) == ARG and disp(off=None) == ARG and disp(E_=-1) == ARG
    assert disp(x=A + 1) == ALIGN and disp(rows=B + 2, elem=1) == ALIGN
    assert disp(rows=A + 32) == OVERLAP and disp(rows=C) == OVERLAP and disp(rows=D - 64) == OVERLAP
    assert lib.msr_dispatch_grad(A, None, C, 10, 2, 16, 0, None) == ARG
    assert lib.msr_dispatch_grad(A, A + 64, C, 10, 2, 16, 0, None) == OVERLAP
    assert lib.msr_combine(A, B, None, C, 10, 2, 16, 0, 0, None) == ARG
    assert lib.msr_combine(A, B, D, C, 10, 2, 16, 0, 9, None) == ARG
    assert lib.msr_combine(A, B + 2, D, C, 10, 2, 16, 0, 1, None) == ALIGN
    assert lib.msr_combine(A, B, B + 16, C, 10, 2, 16, 0, 1, None) == OVERLAP
    grad = lambda dy=A, rows=B, w=C, dr=D, dw=E, pos=W, off=W + 4096: lib.msr_combine_grad(  # noqa: E731
        dy, 16, rows, w, dr, dw, pos, off, 8, 10, 2, 16, 0, 1, None)
    assert grad(dr=None, dw=None) == 0
    assert grad(dy=None) == ARG and grad(rows=None) == ARG and grad(w=None) == ARG and grad(off=None) == ARG
    assert grad(dw=E + 2) == ALIGN
    assert grad(dr=B) == OVERLAP and grad(dw=C) == OVERLAP and grad(dr=D, dw=D + 8) == OVERLAP


def test_products(lib):
    fwd = lambda x=A, ldx=64, w=B, y=C, off=D, rows=100, E_=4, i=64, o=32: lib.msr_experts_forward(  # noqa: E731
        x, ldx, w, y, off, rows, E_, i, o, None)
    assert fwd(rows=0) == 0
    assert fwd(rows=-1) == ARG and fwd(rows=1 << 30) == ARG and fwd(E_=0) == ARG and fwd(E_=1025) == ARG
    assert fwd(i=60, ldx=64) == ARG and fwd(o=33) == ARG and fwd(i=1 << 16, o=1 << 15, ldx=1 << 16) == ARG
    assert fwd(ldx=63) == ARG and fwd(ldx=1 << 22) == ARG and fwd(x=None) == ARG and fwd(off=None) == ARG
    assert fwd(y=1 << 50, rows=(1 << 30) - 1, o=1 << 14) == ARG and b"tiles" in lib.msr_last_error()
    assert fwd(x=A + 8) == ALIGN and fwd(ldx=68) == ALIGN and fwd(off=D + 2) == ALIGN
    assert fwd(y=A + 128) == OVERLAP and fwd(y=B + 16) == OVERLAP and fwd(y=D - 64) == OVERLAP
    assert lib.msr_experts_dgrad(A, 31, B, C, D, 100, 4, 64, 32, None) == ARG
    assert lib.msr_experts_wgrad(C, A, 64, B, 24, D, 100, 4, 64, 32, None) == ARG
    assert lib.msr_experts_wgrad(A, A, 64, B, 32, D, 100, 4, 64, 32, None) == OVERLAP
    acc = lambda mode, inject=None: lib.msr_experts_wgrad_sr_accum(C, A, 64, B, 32, D, 100, 4, 64, 32, 7, 0, mode, inject, None)  # noqa: E731
    assert acc(3) == ARG and acc(-1) == ARG and acc(2) == ARG
    t, split = ctypes.c_int32(), ctypes.c_int32()
    assert lib.msr_experts_tile(4, 100, 4, 64, 32, ctypes.byref(t), ctypes.byref(split)) == ARG
    for product in range(4):
        for rows, E_, i, o in ((1, 1, 8, 8), (61, 8, 256, 512), (32768, 8, 4096, 14336), (1 << 29, 1024, 1024, 1 << 19)):
            assert lib.msr_experts_tile(product, rows, E_, i, o, ctypes.byref(t), ctypes.byref(split)) == 0
            assert t.value in (64, 128, 256) and split.value in (0, 1)


def test_python_needs_a_gpu_and_fitting_arguments(lib):
    import muon_sr_amd as M
    g = torch.zeros(4, dtype=torch.bfloat16)
    for call in (lambda: M.grad_norm([g]), lambda: M.clip_grads([g], 1.0), lambda: M.grad_norm([g], 0.5),
                 lambda: M.order_tokens(torch.zeros((2, 2), dtype=torch.int64), 4), lambda: M.clip_grads([g, g], 1.0, out=[g])):
        with pytest.raises(ValueError):
            call()
    assert M.grad_norm([]).item() == 0.0 and M.clip_grad_norm_([], 1.0).item() == 0.0
    layer = M.SRExperts(3, 16, 24)
    assert layer.weight.shape == (3, 24, 16) and layer.weight.dtype == torch.bfloat16
    assert layer.weight.abs().max() <= 1 / math.sqrt(16)
    with pytest.raises(ValueError, match="GPU"):
        layer(torch.zeros((2, 16), dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32))


def test_the_norms_workspace_does_not_grow_with_the_list(lib):
    """Every work-group of a clip launch adds up all partial sums: they stay at one per work-group of a launch."""
    size = ctypes.c_size_t()
    for tensors in (1, 113, 1000, 9000):
        assert lib.msr_grad_norm_workspace_bytes(*items(*[(A + (i << 24), 0, 1 << 22, 0) for i in range(tensors)]),
                                                 ctypes.byref(size)) == 0
        assert 8 <= size.value <= 8 * 4096


def test_clip_grad_norm_takes_the_arguments_of_torchs():
    import inspect
    import muon_sr_amd as M
    want, got = (list(inspect.signature(f).parameters.values()) for f in (torch.nn.utils.clip_grad_norm_, M.clip_grad_norm_))
    assert [(p.name, p.default) for p in got] == [(p.name, p.default) for p in want]
    assert M.clip_grad_norm_([], 1.0, foreach=True).item() == 0.0
