"""The embedding, norm, router's balance loss and head together, as a training step calls them: against the formula in 64 bits, with a
weight that the embedding and the head share, on other streams and threads, in HIP graphs, and under saved-tensor hooks."""
import importlib.util
import math
import os
import random
import threading

import pytest
import torch

from _gpu import DEV, ROOT, check, need_gpu, stream

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
U, H = 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope="module", autouse=True)
def L():
    return need_gpu()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def inputs(seed, n=700, vocab=1300, d=136, experts=12):
    g = gen(seed)
    r = lambda *s, k=1.0: torch.randn(s, generator=g, device=DEV).mul_(k).to(BF16)  # noqa: E731
    ids = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    target = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    target[::9] = -100
    return dict(ids=ids, target=target, mask=target != -100, table=r(vocab, d, k=0.3), w=r(d, k=0.1) + 1, b=r(d, k=0.1), router=r(experts, d, k=0.2),
                head=r(vocab, d, k=2.0 / math.sqrt(d)))


LEAVES = ("table", "w", "b", "router", "head")


def step(t):
    """Loss, counts and every gradient of one step of the operators."""
    from muon_sr_amd import balance_loss, embedding, layer_norm, linear_cross_entropy
    p = {k: t[k].detach().requires_grad_(True) for k in LEAVES}
    x = embedding(t["ids"], p["table"], scale=2.0)
    h = layer_norm(x, p["w"], p["b"])
    logits = h @ p["router"].t()
    chosen = torch.topk(logits.float(), 2, dim=1).indices
    balance, counts = balance_loss(logits, chosen, t["mask"])
    y = h + x
    loss = linear_cross_entropy(layer_norm(y, p["w"], p["b"]), p["head"], t["target"])
    return [loss.detach(), balance.detach(), counts, *torch.autograd.grad(loss + 0.1 * balance, [p[k] for k in LEAVES])]


def test_step_against_its_formula():
    """Between the operators values are rounded to bf16 (relative error up to 2^-8, 2^-9 in the mean): x, h, router's logits, y, the second
    norm's output and G on the way, and as many gradients on the way back; the norm of the error of any result stays below 12 of
    the mean ones, 2.4e-2 of its own."""
    t = inputs(1)
    got = step(t)
    p = {k: t[k].double().requires_grad_(True) for k in LEAVES}
    norm = lambda v: torch.nn.functional.layer_norm(v, v.shape[-1:], p["w"], p["b"], 1e-5)  # noqa: E731
    x = 2.0 * p["table"][t["ids"]]
    h = norm(x)
    logits = h @ p["router"].t()
    share = got[2].double() / (2 * t["mask"].sum())
    balance = 12 * (share * torch.softmax(logits, 1)[t["mask"]].mean(0)).sum()
    S = norm(h + x) @ p["head"].t()
    loss = torch.nn.functional.cross_entropy(S, t["target"])
    want = torch.autograd.grad(loss + 0.1 * balance, [p[k] for k in LEAVES])
    assert int(got[2].sum()) == 2 * int(t["mask"].sum())
    for a, b in zip([*got[:2], *got[3:]], [loss.detach(), balance.detach(), *want]):
        assert torch.linalg.norm(a.double() - b) <= 2.4e-2 * torch.linalg.norm(b)


def test_shared_weight(L):
    """A weight that the embedding and the head share: the head's gradient reaches the accumulator first, then the embedding's, each with
    its own seed; both are what the stored gradients and msr_sr_accum give."""
    import muon_sr_amd as M
    from muon_sr_amd import _lib
    vocab, d, n = 900, 72, 500
    table, head = M.SREmbedding(vocab, d, device=DEV), M.SRHead(d, vocab, device=DEV)
    head.weight = table.weight
    g = gen(2)
    want = None
    for micro in range(2):
        ids = torch.randint(0, vocab, (n,), generator=g, device=DEV)
        target = torch.randint(0, vocab, (n,), generator=g, device=DEV)
        random.seed(micro)
        seeds = [random.getrandbits(32) for _ in range(2)]
        random.seed(micro)
        head.loss(table(ids), target).backward()
        w = table.weight.detach().requires_grad_(True)
        x = M.embedding(ids, w).detach().requires_grad_(True)
        dx, dhead = torch.autograd.grad(M.linear_cross_entropy(x, w, target), (x, w))
        dtable, = torch.autograd.grad(M.embedding(ids, w), w, dx)
        first, want = want is None, torch.empty_like(dhead) if want is None else want
        for k, dw in enumerate((dhead, dtable)):
            before = want.clone()
            check(L, L.msr_sr_accum(want.data_ptr(), dw.data_ptr(), 0, dw.numel(), seeds[k], int(first and k == 0), _lib.noise_mode(), None, stream()))
            if k == 1:
                missed = torch.ones(vocab, dtype=torch.bool, device=DEV)
                missed[ids] = False
                want[missed] = before[missed]
        assert table.weight.grad is None and torch.equal(table.weight.acc_grad, want)


def test_another_stream():
    t = inputs(3)
    want = step(t)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(t)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_threads_at_once():
    """Two threads, a stream each, different inputs: each gets its own results."""
    ts = [inputs(4), inputs(5, n=1100, vocab=700, d=64)]
    want = [step(t) for t in ts]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            for _ in range(20):
                got = step(ts[k])
                side.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(want[k], got)):
                    bad.append(k)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not bad and not any(t.is_alive() for t in threads)


def test_graph_replays():
    """Two steps of different sizes captured, replayed in turn on other inputs with eager work in between: each replay is the eager
    result."""
    static = [inputs(6), inputs(7, n=300, vocab=5000, d=64)]
    graphs, outs = [], []
    for t in static:
        step(t)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(t))
        graphs.append(g)
    for seed in (8, 9, 10):
        other = [inputs(seed), inputs(seed + 20, n=300, vocab=5000, d=64)]
        for t, o in zip(static, other):
            for k in t:
                t[k].copy_(o[k])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out, o in zip(outs, other):
            want = step(o)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def direct(f, *args):
    return f(*args)


def checkpointed(f, *args):
    return torch.utils.checkpoint.checkpoint(f, *args, use_reentrant=False)


def offloaded(f, *args):
    with torch.autograd.graph.save_on_cpu():
        return f(*args)


def turned(f, *args):
    """Tensors come back with their last dimension of the largest stride, vectors with gaps."""
    def columns(t):
        if t.dim() == 0:
            return t
        return torch.stack([t, t], 1)[:, 0] if t.dim() == 1 else t.transpose(-1, -2).contiguous().transpose(-1, -2)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), columns):
        return f(*args)


@pytest.mark.parametrize("way", [checkpointed, offloaded, turned], ids=lambda f: f.__name__)
def test_saved_tensors(way):
    """Gradients under saved-tensor hooks equal those without, bit for bit."""
    from muon_sr_amd import balance_loss, embedding, layer_norm, linear_cross_entropy
    t = inputs(11)
    chosen = torch.randint(0, 12, (700, 2), generator=gen(12), device=DEV)

    def model(table, w, b, router, head):
        h = layer_norm(embedding(t["ids"], table), w, b)
        balance, _ = balance_loss(h @ router.t(), chosen, t["mask"])
        return linear_cross_entropy(h, head, t["target"]) + balance

    results = []
    for how in (direct, way):
        leaves = [t[k].clone().requires_grad_(True) for k in LEAVES]
        loss = how(model, *leaves)
        results.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("way", [checkpointed, offloaded, turned], ids=lambda f: f.__name__)
def test_accumulators_under_saved_tensor_hooks(way):
    """The accumulators are the parameters' under hooks too, with the same bits."""
    import muon_sr_amd as M
    t = inputs(13)
    table, head = M.SREmbedding(1300, 136, device=DEV), M.SRHead(136, 1300, device=DEV)
    results = []
    for how in (direct, way):
        random.seed(5)
        for _ in range(2):
            how(lambda ids: head.loss(table(ids), t["target"]), t["ids"]).backward()
        results.append([m.weight.acc_grad for m in (table, head)])
        assert table.weight.grad is None and head.weight.grad is None
        del table.weight.acc_grad, head.weight.acc_grad
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_frozen_and_evaluated():
    """No gradient, no accumulator: frozen weights, and evaluation."""
    import muon_sr_amd as M
    t = inputs(14)
    table, head = M.SREmbedding(1300, 136, device=DEV), M.SRHead(136, 1300, device=DEV)
    with torch.no_grad():
        loss = head.loss(table(t["ids"]), t["target"])
    assert not loss.requires_grad
    table.weight.requires_grad_(False)
    head.weight.requires_grad_(False)
    x = table(t["ids"]).requires_grad_(True)
    assert torch.equal(head.loss(x, t["target"]), loss)
    dx, = torch.autograd.grad(head.loss(x, t["target"]), x)
    assert dx.shape == x.shape and not hasattr(head.weight, "acc_grad") and not hasattr(table.weight, "acc_grad")


def test_errors_keep_their_type():
    """What the library refuses is MuonSRLibraryError, from the nodes and from the module."""
    import muon_sr_amd as M
    from muon_sr_amd._lib import MuonSRLibraryError
    t = inputs(15)
    flat = torch.zeros(1300 * 136 + 1, dtype=BF16, device=DEV)
    with pytest.raises(MuonSRLibraryError, match="aligned"):
        M.linear_cross_entropy(t["table"][t["ids"]], flat[1:].view(1300, 136), t["target"])
    with pytest.raises(MuonSRLibraryError, match="aligned"):
        M.SRHead.loss(_holding(flat[1:].view(1300, 136)), t["table"][t["ids"]], t["target"])


class _holding:
    def __init__(self, weight):
        self.weight = torch.nn.Parameter(weight)


def test_second_derivatives_are_refused():
    from muon_sr_amd import balance_loss, embedding, layer_norm, linear_cross_entropy
    t = inputs(16)
    chosen = torch.zeros((700, 2), dtype=torch.int64, device=DEV)
    calls = [lambda v: linear_cross_entropy(v, t["head"], t["target"]), lambda v: layer_norm(v, t["w"], t["b"]).float().square().mean(),
             lambda v: balance_loss(v[:, :12], chosen)[0]]
    for f in calls:
        x = t["table"][t["ids"]].detach().requires_grad_(True)
        dx, = torch.autograd.grad(f(x), x, create_graph=True)
        with pytest.raises(RuntimeError, match="derivative"):
            dx.float().square().sum().backward()
    w = t["table"].clone().requires_grad_(True)
    dw, = torch.autograd.grad(embedding(t["ids"], w).float().square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="derivative"):
        dw.float().square().sum().backward()


def test_example_uses_them():
    spec = importlib.util.spec_from_file_location("moe_train", os.path.join(ROOT, "examples", "moe_train.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    torch.manual_seed(0)
    model = m.Model(d=64, hidden=96, experts=4, blocks=1)
    window = torch.randint(0, 256, (300, 5), generator=gen(17), device=DEV)
    loss, balance = model.loss(window[:, :4], window[:, 4])
    (loss + 0.01 * balance).backward()
    assert model.embed.weight.acc_grad.shape == (256, 64) and model.head.weight.acc_grad.shape == (256, 64)
    assert model.norms[0].weight.grad.shape == (64,) and model.moe[0].router.weight.grad.any()
    logits, _ = model(window[:, :4])
    # the logits that torch gives are rounded to bf16, 2^-8 of up to their largest
    want = torch.nn.functional.cross_entropy(logits.double(), window[:, 4])
    assert abs(loss.item() - want.item()) <= 2 * H * logits.abs().max().item() + 1e-5


def shifted(f, *args):
    """Tensors come back one element behind the start of their memory, as those of a buffer that they share."""
    def behind(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), behind):
        return f(*args)


def test_saved_tensors_of_a_shared_buffer():
    """Such hooks change no bit, and refuse nothing, with the accumulators and without."""
    test_saved_tensors(shifted)
    test_accumulators_under_saved_tensor_hooks(shifted)


def test_transforms_and_forward_mode_are_refused():
    """torch.func's transforms and forward-mode derivatives raise; none returns without a derivative."""
    from torch.autograd import forward_ad
    from muon_sr_amd import balance_loss, embedding, layer_norm, linear_cross_entropy
    t = inputs(18)
    chosen = torch.zeros((700, 2), dtype=torch.int64, device=DEV)
    x = t["table"][t["ids"]]
    calls = [(lambda v: linear_cross_entropy(v, t["head"], t["target"]), x), (lambda v: linear_cross_entropy(x, v, t["target"]), t["head"]),
             (lambda v: layer_norm(v, t["w"], t["b"]), x), (lambda v: layer_norm(x, v, t["b"]), t["w"]), (lambda v: embedding(t["ids"], v), t["table"]),
             (lambda v: balance_loss(v, chosen)[0], torch.zeros((700, 12), device=DEV))]
    for f, v in calls:
        for transform in (lambda: torch.func.grad(lambda z: f(z).float().sum())(v), lambda: torch.func.vmap(f)(torch.stack([v, v])),
                          lambda: torch.func.jvp(f, (v,), (v,))):
            with pytest.raises(RuntimeError, match="functorch"):
                transform()
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="jvp"):
            f(forward_ad.make_dual(v, v))
