"""The operators together: a mixture-of-experts layer against its formula in 64 bits, on another stream, in a
HIP graph, and a short training run."""
import importlib.util
import math
import os

import pytest
import torch

from _gpu import DEV, ROOT, need_gpu

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def example():
    need_gpu()
    spec = importlib.util.spec_from_file_location("moe_train", os.path.join(ROOT, "examples", "moe_train.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rel(x, ref):
    return (torch.linalg.norm(x.double() - ref) / torch.linalg.norm(ref)).item()


def make_layer(example, d=64, hidden=96, experts=5, k=2):
    torch.manual_seed(3)
    layer = example.MoE(d, hidden, experts, k, DEV)
    x = torch.randn((301, d), generator=gen(1), device=DEV, dtype=BF16)
    dy = torch.randn((301, d), generator=gen(2), device=DEV, dtype=BF16)
    return layer, x, dy


def test_layer_against_its_formula(example):
    """Output and gradients of a layer against the dense formula in 64 bits with the same choice of experts.
    Between the operators values are rounded to bf16 (relative error up to 2^-8, 2^-9 in the mean) five times on
    the way forward (rows are copies; up, gelu, down, the sum; scores) and five on the way back: the norm of the
    error of any result is below 10 * 2^-9 = 2e-2 of its own."""
    layer, x, dy = make_layer(example)
    x.requires_grad_(True)
    y, _ = layer(x)
    y.backward(dy)
    ids = torch.topk(torch.softmax(layer.router(x).float(), -1), 2, dim=-1).indices
    X = x.detach().double().requires_grad_(True)
    R, U, D = (w.detach().double().requires_grad_(True) for w in (layer.router.weight, layer.up.weight, layer.down.weight))
    scores = torch.softmax(X @ R.t(), -1).gather(1, ids)
    weights = scores / scores.sum(-1, keepdim=True)
    Y = 0.0
    for j in range(2):
        h = torch.nn.functional.gelu((U[ids[:, j]] @ X.unsqueeze(2)).squeeze(2))
        Y = Y + weights[:, j:j + 1] * (D[ids[:, j]] @ h.unsqueeze(2)).squeeze(2)
    Y.backward(dy.double())
    assert rel(y.detach(), Y.detach()) < 2e-2
    assert rel(x.grad, X.grad) < 2e-2
    assert rel(layer.router.weight.grad, R.grad) < 2e-2
    # accumulated from zero: one stochastic rounding more (2^-8 at most)
    assert rel(layer.up.weight.acc_grad, U.grad) < 2e-2 and rel(layer.down.weight.acc_grad, D.grad) < 2e-2


def chain(ids, x, w, up, dy, outs):
    """Every operator once, on tensors only."""
    from muon_sr_amd import clip_grads, combine_tokens, dispatch_tokens, expert_linear, order_tokens
    order = order_tokens(ids, up.shape[0])
    rows = dispatch_tokens(x, order)
    y = combine_tokens(expert_linear(rows, up, order.offsets), w, order)
    grads = torch.autograd.grad(y, (x, w, up), dy)
    norm = clip_grads([grads[0], grads[2]], 0.5, out=outs)
    return (*order, rows, y, *grads, norm, *outs)


def chain_inputs(seed):
    g = gen(seed)
    r = lambda *s: torch.randn(s, generator=g, device=DEV, dtype=BF16)  # noqa: E731
    ids = torch.randint(-1, 6, (20000, 2), generator=g, device=DEV)
    return [ids, r(20000, 128), torch.rand((20000, 2), generator=g, device=DEV), r(6, 264, 128) * 0.1, r(20000, 264)]


def run_chain(t):
    t = [v if v.dtype == torch.int64 else v.detach().requires_grad_(True) for v in t]
    outs = [torch.empty((20000, 128), dtype=BF16, device=DEV), torch.empty((6, 264, 128), dtype=BF16, device=DEV)]
    return chain(*t[:4], t[4].detach(), outs)


def test_another_stream():
    need_gpu()
    inputs = chain_inputs(5)
    want = run_chain(inputs)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run_chain(inputs)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_graph_replays():
    """Captured once, replayed on other inputs with eager work in between: each replay is the eager result."""
    need_gpu()
    static = chain_inputs(6)
    run_chain(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run_chain(static)
    for seed in (7, 8, 9, 10):
        inputs = chain_inputs(seed)
        for s, i in zip(static, inputs):
            s.copy_(i)
        graph.replay()
        torch.cuda.synchronize()
        want = run_chain(inputs)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_training_run(example):
    """The example for 60 steps: from the uniform loss (ln 256 = 5.5) to below 3.2, with a finite norm each step."""
    losses, norms = example.train(steps=60, micro=2, tokens=2048)
    assert all(math.isfinite(v) for v in losses + norms)
    assert losses[0] > 5.0 and sum(losses[-10:]) / 10 < 3.2
