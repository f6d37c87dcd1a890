"""Where the weight gradients of SRExperts and SRLinear go, without a GPU: their autograd functions with the
products stubbed, and a library whose accumulations mark the buffer that they are given."""
import ctypes

import pytest
import torch

BF16 = torch.bfloat16
MARK = 0x3f                        # bf16 0x3f3f = 0.7461


class Library:
    """The two accumulation entry points: they fill the buffer with MARK, or refuse with `status`."""

    def __init__(self):
        self.calls, self.status = [], 0

    def _accumulate(self, acc, numel, zero_init):
        self.calls.append(zero_init)
        if not self.status:
            ctypes.memset(acc, MARK, 2 * numel)
        return self.status

    def msr_experts_wgrad_sr_accum(self, acc, x, ldx, dy, lddy, offsets, rows, experts, i, o, seed, zero_init, *rest):
        return self._accumulate(acc, experts * i * o, zero_init)

    def msr_linear_wgrad_sr_accum(self, acc, x, ldx, dy, lddy, tokens, i, o, seed, zero_init, *rest):
        return self._accumulate(acc, i * o, zero_init)

    def msr_last_error(self):
        return b"refused"


@pytest.fixture
def library(monkeypatch):
    from muon_sr_amd import _lib, experts, linear
    L = Library()
    monkeypatch.setattr(_lib, "lib", lambda: L)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(experts, "_one_gpu", lambda *a: None)
    monkeypatch.setattr(experts, "_forward", lambda x, w, off: x @ w[0].t())
    monkeypatch.setattr(experts, "_dgrad", lambda dy, w, off: dy @ w[0])
    monkeypatch.setattr(experts, "_wgrad", lambda w, x, dy, off: (dy.t() @ x).unsqueeze(0))
    monkeypatch.setattr(linear, "_fits", lambda weight, x, dy: True)
    return L


def make_experts():
    from muon_sr_amd import SRExperts
    layer, offsets = SRExperts(1, 16, 24), torch.tensor([0, 5], dtype=torch.int32)
    return layer, lambda x: layer(x, offsets)


def make_linear():
    from muon_sr_amd import SRLinear
    layer = SRLinear(16, 24, bias=False, dtype=BF16)
    return layer, layer


def plain(f, x):
    return f(x)


def checkpoint(f, x):
    return torch.utils.checkpoint.checkpoint(f, x, use_reentrant=False)


def reentrant(f, x):
    return torch.utils.checkpoint.checkpoint(f, x, use_reentrant=True)


def hooks(f, x):
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t):
        return f(x)


def on_cpu(f, x):
    with torch.autograd.graph.save_on_cpu():
        return f(x)


MAKERS = [make_experts, make_linear]
WAYS = [plain, checkpoint, reentrant, hooks, on_cpu]
named = pytest.mark.parametrize("make", MAKERS, ids=lambda f: f.__name__)


@named
@pytest.mark.parametrize("way", WAYS, ids=lambda f: f.__name__)
def test_the_parameter_holds_the_accumulator(library, make, way):
    layer, f = make()
    for micro in range(2):
        x = torch.randn(5, 16, dtype=BF16, requires_grad=True)
        way(f, x).sum().backward()
        assert x.grad is not None
    assert library.calls == [1, 0]
    assert layer.weight.grad is None and bool((layer.weight.acc_grad.view(torch.int16) == MARK * 257).all())


@named
def test_a_weight_that_is_computed_returns_its_gradient(library, make):
    """A parametrized weight is another tensor in every forward pass: its gradient goes through autograd."""
    class Double(torch.nn.Module):
        def forward(self, w):
            return 2 * w

    layer, f = make()
    torch.nn.utils.parametrize.register_parametrization(layer, "weight", Double())
    x = torch.randn(5, 16, dtype=BF16)
    f(x).backward(torch.ones(5, 24, dtype=BF16))
    grad = layer.parametrizations.weight.original.grad
    assert library.calls == [] and torch.equal(grad.view(24, 16), 2 * (torch.ones(24, 5, dtype=BF16) @ x))


def accumulate_experts(weight, seed=5):
    from muon_sr_amd import experts_wgrad_sr_accum
    x, dy = torch.zeros(5, 16, dtype=BF16), torch.zeros(5, 24, dtype=BF16)
    experts_wgrad_sr_accum(weight, x, dy, torch.tensor([0, 5], dtype=torch.int32), seed=seed)


def accumulate_linear(weight, seed=5):
    from muon_sr_amd import linear_wgrad_sr_accum
    assert linear_wgrad_sr_accum(weight, torch.zeros(5, 16, dtype=BF16), torch.zeros(5, 24, dtype=BF16), seed=seed)


CALLS = [(accumulate_experts, (1, 24, 16)), (accumulate_linear, (24, 16))]
called = pytest.mark.parametrize("call,shape", CALLS, ids=[c.__name__ for c, _ in CALLS])


@called
def test_a_buffer_that_is_no_accumulator_is_refused(library, call, shape):
    """Another type, order, size or device than the kernel writes."""
    weight = torch.nn.Parameter(torch.zeros(shape, dtype=BF16))
    turned = torch.zeros(shape, dtype=BF16).transpose(-1, -2).contiguous().transpose(-1, -2)
    smaller = torch.zeros(shape, dtype=BF16)[..., :8].contiguous()
    for buffer in (torch.zeros(shape), turned, smaller, torch.zeros(24 * 16, dtype=BF16),
                   torch.zeros(shape, dtype=BF16, device="meta"), None):
        weight.acc_grad = buffer
        with pytest.raises(ValueError, match="acc_grad"):
            call(weight)
        assert library.calls == [] and weight.acc_grad is buffer
    weight.acc_grad = torch.zeros(shape, dtype=BF16)
    call(weight)
    assert library.calls == [0]


@called
def test_a_refused_first_call_leaves_no_accumulator(library, call, shape):
    from muon_sr_amd import _lib
    weight = torch.nn.Parameter(torch.zeros(shape, dtype=BF16))
    library.status = 1005
    with pytest.raises(_lib.MuonSRLibraryError, match="refused"):
        call(weight)
    assert not hasattr(weight, "acc_grad")
    library.status = 0
    call(weight)
    call(weight)
    assert library.calls == [1, 1, 0] and weight.acc_grad.shape == shape
