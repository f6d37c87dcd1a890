"""Saved-tensor hooks may give a tensor back in another memory layout (the same values, type and device): what the
backward passes of the token and experts operators then hand to the library, without a GPU."""
import ctypes

import pytest
import torch

BF16 = torch.bfloat16


def memory(address, shape):
    """A copy of a row-major bf16 matrix at an address."""
    n = torch.Size(shape).numel()
    return torch.frombuffer(bytearray(ctypes.string_at(address, 2 * n)), dtype=BF16).view(shape)


def fill(address, values):
    ctypes.memmove(address, values.contiguous().data_ptr(), 2 * values.numel())


class Library:
    """The entry points on host memory, in torch."""

    def msr_combine(self, *a):
        return 0

    def msr_combine_grad(self, dy, lddy, rows, w, drows, dw, position, offsets, experts, tokens, k, d, elem, welem, stream):
        self.rows, self.w = memory(rows, (tokens * k, d)), memory(w, (tokens, k))
        fill(drows, memory(rows, (tokens * k, d)))
        fill(dw, memory(w, (tokens, k)))
        return 0

    def msr_experts_forward(self, *a):
        return 0

    def msr_experts_dgrad(self, dy, lddy, w, dx, offsets, rows, experts, i, o, stream):
        self.w, self.offsets = memory(w, (experts, o, i)), ctypes.string_at(offsets, 4 * (experts + 1))
        return 0

    def msr_experts_wgrad(self, dw, x, ldx, dy, lddy, offsets, rows, experts, i, o, stream):
        self.x = torch.stack([memory(x + 2 * ldx * r, (i,)) for r in range(rows)])
        return 0

    def msr_experts_wgrad_sr_accum(self, acc, x, ldx, dy, lddy, offsets, rows, experts, i, o, *rest):
        return self.msr_experts_wgrad(acc, x, ldx, dy, lddy, offsets, rows, experts, i, o, None)


@pytest.fixture
def library(monkeypatch):
    from muon_sr_amd import _lib, experts
    L = Library()
    monkeypatch.setattr(_lib, "lib", lambda: L)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(experts, "_one_gpu", lambda *a: None)
    return L


def columns(t):
    """t with its last dimension of the largest stride; a vector with gaps."""
    if t.dim() == 1:
        return torch.stack([t, t], 1)[:, 0]
    return t.transpose(-1, -2).contiguous().transpose(-1, -2)


def turned():
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, columns)


def randn(*shape):
    return torch.randn(shape, dtype=BF16).requires_grad_(True)


def test_combine(library):
    from muon_sr_amd import TokenOrder, combine_tokens
    order = TokenOrder(torch.tensor([0, 6], dtype=torch.int32), torch.arange(6, dtype=torch.int32).view(3, 2),
                       torch.arange(6, dtype=torch.int32))
    rows, w = randn(6, 16), randn(3, 2)
    with turned():
        y = combine_tokens(rows, w, order)
    y.backward(torch.ones(3, 16, dtype=BF16))
    assert torch.equal(library.rows, rows.detach()) and torch.equal(library.w, w.detach())
    assert torch.equal(rows.grad, rows.detach()) and torch.equal(w.grad, w.detach())   # (what the stub writes)


def test_expert_linear(library):
    from muon_sr_amd import SRExperts, expert_linear
    x, w, offsets = randn(5, 16), randn(2, 24, 16), torch.tensor([0, 3, 5], dtype=torch.int32)
    layer = SRExperts(2, 16, 24)
    for weight, run in ((w, lambda: expert_linear(x, w, offsets)), (layer.weight, lambda: layer(x, offsets))):
        with turned():
            y = run()
        y.backward(torch.ones(5, 24, dtype=BF16))
        assert torch.equal(library.w, weight.detach()) and torch.equal(library.x, x.detach())
        assert library.offsets == offsets.numpy().tobytes()
