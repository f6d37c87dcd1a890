"""Gradients under saved-tensor hooks (activation checkpointing, offloading to the host, tensors that come back in
another layout) equal those without, bit for bit: the same kernels on the same values."""
import random

import pytest
import torch

from _gpu import DEV, need_gpu

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def L():
    return need_gpu()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(shape, seed, dtype=BF16):
    return torch.randn(shape, generator=gen(seed), device=DEV).to(dtype)


def direct(f, *args):
    return f(*args)


def checkpointed(f, *args):
    return torch.utils.checkpoint.checkpoint(f, *args, use_reentrant=False)


def offloaded(f, *args):
    with torch.autograd.graph.save_on_cpu():
        return f(*args)


def hooked(f, *args):
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t):
        return f(*args)


HOOKS = pytest.mark.parametrize("way", [checkpointed, offloaded, hooked], ids=lambda f: f.__name__)


def accumulated(layer, f, way):
    """The accumulator and the input gradients of three micro-batches, from the same random state."""
    random.seed(11)
    dxs = []
    for micro in range(3):
        x = randn((189, layer.weight.shape[-1]), micro).requires_grad_(True)
        way(f, x).backward(randn((189, layer.weight.shape[-2]), 10 + micro))
        dxs.append(x.grad)
    acc = layer.weight.acc_grad
    del layer.weight.acc_grad
    assert layer.weight.grad is None
    return [acc, *dxs]


@HOOKS
def test_experts_accumulate(way):
    from muon_sr_amd import SRExperts
    layer = SRExperts(4, 64, 48, device=DEV)
    offsets = torch.tensor([0, 100, 100, 160, 187], dtype=torch.int32, device=DEV)
    f = lambda x: layer(x, offsets)  # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(accumulated(layer, f, direct), accumulated(layer, f, way)))


@HOOKS
def test_linear_accumulates(way):
    from muon_sr_amd import SRLinear
    layer = SRLinear(256, 512, bias=False, device=DEV, dtype=BF16)
    f = lambda x: layer(torch.cat([x, x[:67]]))  # noqa: E731   (256 tokens)
    cut = lambda x: f(x)[:189]  # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(accumulated(layer, cut, direct), accumulated(layer, cut, way)))


def turned(f, *args):
    """Tensors come back with their last dimension of the largest stride, vectors with gaps."""
    def columns(t):
        return torch.stack([t, t], 1)[:, 0] if t.dim() == 1 else t.transpose(-1, -2).contiguous().transpose(-1, -2)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, columns):
        return f(*args)


@pytest.mark.parametrize("way", [checkpointed, offloaded, hooked, turned], ids=lambda f: f.__name__)
def test_layer_of_operators(way):
    """dispatch, the experts' products and combine: every input's gradient."""
    from muon_sr_amd import combine_tokens, dispatch_tokens, expert_linear, order_tokens
    ids = torch.randint(-1, 5, (301, 2), generator=gen(1), device=DEV)
    tensors = [randn((301, 72), 2), torch.rand((301, 2), generator=gen(3), device=DEV), randn((5, 136, 72), 4), randn((5, 72, 136), 5)]
    dy = randn((301, 72), 6)

    def layer(x, w, up, down):
        order = order_tokens(ids, 5)
        rows = expert_linear(dispatch_tokens(x, order), up, order.offsets)
        return combine_tokens(expert_linear(rows, down, order.offsets), w, order)

    results = []
    for how in (direct, way):
        leaves = [t.clone().requires_grad_(True) for t in tensors]
        y = how(layer, *leaves)
        results.append([y, *torch.autograd.grad(y, leaves, dy)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
