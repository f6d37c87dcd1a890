"""The head's loss and gradients against 64-bit evaluations of their definition on the same bf16 operands.

Bounds, with u = 2^-24 (an fp32 rounding) and h = 2^-8 (a bf16 one).  A logit S formed in fp32 from d products is off by at
most eS = 2 (d + 1) u sum|x w| (the factor 2: any order of the sums, and what higher terms add).  exp of an argument
a = x - m costs 4 u (|a| + 1) + 2 u |m| at most: its product with log2 e, that constant, the difference and the function.  The sum behind l has at most depth =
64 + vocab / 64 additions one after the other (32 in a lane, the waves', and a share of the tiles), so l is off by at most
el = max eS + 2 depth u + 8 u (|l| + 1) + 2 u max|S|, and the loss by eS + el + u |loss|.
G = g (p - [target]) is off by eG = g (p (eS + el + 4 u (|S - l| + 1) + 2 u |l|) + 2 u), then h |G| by its rounding (a rounding is
off by less than h / (1 + h), which leaves room for the division by c), or h^2 |G| of up to 32 rows (128 where each has its own g), whose G is kept
as two numbers; a product over
K terms adds 2 (K + 16) u sum|terms| (c's product among them) and the stored value's rounding h |value|.  Values below the smallest normal
number may vanish: 2^-126 per term."""
import ctypes
import math
import random

import pytest
import torch

from _gpu import DEV, check, need_gpu, stream

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
U, H = 2.0 ** -24, 2.0 ** -8
REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


@pytest.fixture(scope="module", autouse=True)
def L():
    return need_gpu()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make(rows, vocab, d, seed, ignored=0.2):
    g = gen(seed)
    w = torch.randn((vocab, d), generator=g, device=DEV).mul_(3.0 / math.sqrt(d)).to(BF16)
    target = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    x = torch.randn((rows, d), generator=g, device=DEV).to(BF16) + (2.5 * torch.rand((rows, 1), generator=g, device=DEV)).to(BF16) * w[target]
    target[torch.rand(rows, generator=g, device=DEV) < ignored] = -100
    return x, w, target, torch.rand(rows, generator=g, device=DEV) + 0.25


def exact(x, w, target, dloss, reduction):
    """Values and bounds in 64 bits: loss, dx, dw and theirs."""
    x, w = x.double(), w.double()
    vocab, d = w.shape
    on = target != -100
    x = torch.where(on[:, None], x, 0.0)
    t = target.clamp(min=0)
    S = x @ w.t()
    eS = 2 * (d + 1) * U * (x.abs() @ w.abs().t())
    l = torch.logsumexp(S, 1)
    el = eS.max(1).values + 2 * (64 + vocab / 64) * U + 8 * U * (l.abs() + 1) + 2 * U * S.abs().max(1).values
    St, eSt = (v.gather(1, t[:, None])[:, 0] for v in (S, eS))
    each = torch.where(on, l - St, 0.0)
    e_each = torch.where(on, eSt + el + U * (l - St).abs(), 0.0)
    n = max(1, int(on.sum()))
    g = dloss.double() if reduction == "none" else dloss.double()[:1].expand(len(t)) / (n if reduction == "mean" else 1)
    g = torch.where(on, g, 0.0)[:, None]
    p = torch.exp(S - l[:, None])
    eG = g * (p * (eS + el[:, None] + 4 * U * ((S - l[:, None]).abs() + 1) + 2 * U * l[:, None].abs()) + 2 * U)
    G = p.clone()
    G[torch.arange(len(t), device=DEV), t] -= 1.0
    G *= g
    eG += (H if len(t) > (128 if reduction == "none" else 32) else H * H) * (G.abs() + eG)

    def product(a, ea, b):
        terms = a.abs() @ b.abs()
        v = a @ b
        return v, H * v.abs() + (1 + H) * (ea @ b.abs() + 2 * (a.shape[1] + 16) * U * terms) + a.shape[1] * 2.0 ** -126

    if reduction == "none":
        loss, e_loss = each, e_each
    else:
        k = n if reduction == "mean" else 1
        loss, e_loss = each.sum() / k, e_each.sum() / k + 2 * U * each.sum() / k
    return (loss, e_loss), product(G, eG, w), product(G.t().contiguous(), eG.t().contiguous(), x)


def near(got, want):
    value, bound = want
    assert got.shape == value.shape
    bad = ~((got.double() - value).abs() <= bound + 1e-37)
    assert not bad.any(), (int(bad.sum()), (got.double() - value).abs().max().item(), bound.max().item())


def run(x, w, target, dloss, reduction):
    from muon_sr_amd import linear_cross_entropy
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(x, w, target, reduction=reduction)
    assert loss.dtype == torch.float32
    dx, dw = torch.autograd.grad(loss, (x, w), dloss if reduction == "none" else dloss[0])
    return loss.detach(), dx, dw


def plan(L, rows, vocab, d):
    out = (ctypes.c_int32 * 7)()
    check(L, L.msr_head_plan(rows, vocab, d, out))
    return list(out)


SIZES = [(1, 1, 8), (1, 17, 8), (7, 512, 256), (2, 9001, 64), (65, 130, 72), (300, 1000, 1032), (257, 4099, 136), (1025, 70, 2048),
         (3000, 8192, 64), (2047, 3001, 1024), (16384, 17001, 64), (5000, 777, 264), (129, 20011, 520), (64, 64, 64), (32, 3001, 1032), (31, 70000, 72), (128, 900, 136), (100, 30011, 520), (4096, 8200, 2048)]


@pytest.mark.parametrize("rows,vocab,d", SIZES)
def test_against_64_bits(rows, vocab, d):
    x, w, target, dloss = make(rows, vocab, d, rows + vocab)
    for reduction in REDUCTIONS:
        want = exact(x, w, target, dloss, reduction)
        for got, value in zip(run(x, w, target, dloss, reduction), want):
            near(got, value)


def test_the_sizes_take_every_tile(L):
    """Tiles of 64, 128 and 256, splits and several pieces are among the sizes above."""
    plans = [plan(L, *s) for s in SIZES]
    for i in (0, 1, 2, 4):
        assert {p[i] for p in plans} == {64, 128, 256}, (i, {p[i] for p in plans})
    assert any(p[3] > 1 for p in plans) and any(p[5] > 1 for p in plans)
    assert any(-(-s[1] // p[6]) > 1 for s, p in zip(SIZES, plans))


def test_ignored_rows_reach_nothing():
    """What ignored rows hold, NaN and infinities too, changes no bit of the others' results; their loss and gradient are 0."""
    x, w, target, dloss = make(700, 1500, 96, 3, ignored=0.4)
    off = target == -100
    want = run(x, w, target, dloss, "none")
    dirty = x.clone()
    dirty[off] = torch.tensor([math.nan, math.inf, -math.inf], device=DEV).to(BF16).repeat(32)
    for a, b in zip(run(dirty, w, target, dloss, "none"), want):
        assert torch.equal(a, b)
    assert not want[0][off].any() and not want[1][off].any()


def test_nothing_to_learn_from():
    """No rows, or ignored ones only: loss 0, gradients 0."""
    for rows in (0, 5):
        x, w, target, dloss = make(rows, 300, 64, 4)
        target.fill_(-100)
        for reduction in REDUCTIONS:
            loss, dx, dw = run(x, w, target, torch.ones(max(rows, 1), device=DEV)[:rows if reduction == "none" else None], reduction)
            assert loss.shape == ((rows,) if reduction == "none" else ()) and not loss.any() and not dx.any() and not dw.any()
            assert dx.shape == x.shape and dw.shape == w.shape


def test_targets_that_are_no_word():
    """Their loss is NaN, and so are their row's gradient and the words'; the other rows' losses are as they are."""
    x, w, target, dloss = make(200, 333, 64, 5, ignored=0.1)
    want = run(x, w, target, dloss, "none")[0]
    at = int((target != -100).nonzero()[7])
    for bad in (333, -1, 1 << 40, -(1 << 33)):
        wrong = target.clone()
        wrong[at] = bad
        loss, dx, dw = run(x, w, wrong, dloss, "none")
        assert loss[at].isnan() and dx[at].isnan().all() and dw.isnan().all()
        others = torch.arange(200, device=DEV) != at
        assert torch.equal(loss[others], want[others]) and not dx[others].isnan().any()
        assert run(x, w, wrong, dloss, "mean")[0].isnan()


def test_other_ignore_index_and_int32():
    from muon_sr_amd import linear_cross_entropy
    x, w, target, dloss = make(150, 200, 64, 6, ignored=0.3)
    want = linear_cross_entropy(x, w, target, reduction="none")
    zero = torch.where(target == -100, 7, torch.where(target == 7, 8, target))      # word 7 is ignored
    assert torch.equal(linear_cross_entropy(x, w, zero, ignore_index=7, reduction="none")[target != 7], want[target != 7])
    assert torch.equal(linear_cross_entropy(x, w, target.int(), reduction="none"), want)


def test_extreme_logits():
    """Logits of +-1e4 and more: the loss is the distance to the maximum, nothing overflows; a row of infinite logits is NaN, alone."""
    g = gen(7)
    x = torch.randn((90, 64), generator=g, device=DEV).mul_(300).to(BF16)
    w = torch.randn((500, 64), generator=g, device=DEV).mul_(30).to(BF16)
    target = torch.randint(0, 500, (90,), generator=g, device=DEV)
    dloss = torch.ones(90, device=DEV)
    for got, want in zip(run(x, w, target, dloss, "none"), exact(x, w, target, dloss, "none")):
        near(got, want)
    clean = run(x, w, target, dloss, "none")
    x[3, 5] = math.inf
    loss, dx, _ = run(x, w, target, dloss, "none")
    others = torch.arange(90, device=DEV) != 3
    assert loss[3].isnan() and torch.equal(loss[others], clean[0][others]) and torch.equal(dx[others], clean[1][others])


def test_shapes_strides_and_wanted_gradients():
    from muon_sr_amd import linear_cross_entropy
    x, w, target, dloss = make(132, 257, 64, 8)
    want = run(x, w, target, dloss, "none")
    wide = torch.zeros((132, 200), dtype=BF16, device=DEV)
    wide[:, 3:67] = x
    turned = x.t().contiguous().t()
    for v in (wide[:, 3:67], turned, x.view(11, 12, 64)):
        leaf, word = v.detach().requires_grad_(True), w.clone().requires_grad_(True)
        t = target.view(v.shape[:-1])
        loss = linear_cross_entropy(leaf, word, t, reduction="none")
        assert torch.equal(loss.detach().flatten(), want[0]) and loss.shape == t.shape
        dx, dw = torch.autograd.grad(loss, (leaf, word), dloss.view(t.shape))
        assert torch.equal(dx.reshape(132, 64), want[1]) and torch.equal(dw, want[2]) and dx.shape == v.shape
    one = x[5:6].expand(40, 64)
    assert torch.equal(linear_cross_entropy(one, w, target[:40]), linear_cross_entropy(one.contiguous(), w, target[:40]))
    assert linear_cross_entropy(x[5], w, target[5]).shape == ()
    # only one gradient wanted
    leaf, word = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(leaf, w, target, reduction="none"), leaf, dloss)[0], want[1])
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, word, target, reduction="none"), word, dloss)[0], want[2])
    assert not linear_cross_entropy(x, w, target).requires_grad


@pytest.mark.parametrize("rows,vocab,d", [(7, 512, 256), (2047, 3001, 1024), (300, 1000, 1032), (4096, 8200, 384), (257, 4099, 136), (4096, 8200, 2048)])
def test_one_gradient_is_that_of_both(rows, vocab, d):
    """Each gradient has the same bits when it is wanted alone."""
    from muon_sr_amd import linear_cross_entropy
    x, w, target, dloss = make(rows, vocab, d, 14)
    _, dx, dw = run(x, w, target, dloss, "none")
    leaf, word = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(leaf, w, target, reduction="none"), leaf, dloss)[0], dx)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, word, target, reduction="none"), word, dloss)[0], dw)


@pytest.mark.parametrize("noise", ["philox8", "triton"])
@pytest.mark.parametrize("rows,vocab,d", [(70, 333, 72), (3000, 8192, 64), (1, 40, 8), (16384, 17001, 64), (1025, 70, 2048)])
def test_accumulated_weight_gradient(L, rows, vocab, d, noise):
    """SRHead's accumulator is, bit for bit, what the stored gradient and msr_sr_accum give, over three micro-batches."""
    import muon_sr_amd as M
    from muon_sr_amd import _lib
    head = M.SRHead(d, vocab, device=DEV)
    was = M.get_sr_noise()
    M.set_sr_noise(noise)
    try:
        want = None
        for micro in range(3):
            x, w, target, dloss = make(rows, vocab, d, micro)
            with torch.no_grad():
                head.weight.copy_(w)
            random.seed(micro)
            seed = random.getrandbits(32)
            random.seed(micro)
            leaf = x.clone().requires_grad_(True)
            head.loss(leaf, target).backward(dloss[0])
            _, dx, dw = run(x, w, target, dloss, "mean")
            first = want is None
            want = torch.empty_like(dw) if first else want
            check(L, L.msr_sr_accum(want.data_ptr(), dw.data_ptr(), 0, dw.numel(), seed, int(first), _lib.noise_mode(), None, stream()))
            assert head.weight.grad is None and torch.equal(head.weight.acc_grad, want) and torch.equal(leaf.grad, dx)
    finally:
        M.set_sr_noise(was)


def test_refused_accumulators_and_parametrized_weights():
    import muon_sr_amd as M
    head = M.SRHead(64, 100, device=DEV)
    x, _, target, _ = make(20, 100, 64, 9)
    for bad in (torch.zeros((100, 64), device=DEV), torch.zeros((64, 100), dtype=BF16, device=DEV).t(), None):
        head.weight.acc_grad = bad
        with pytest.raises(ValueError, match="acc_grad"):
            head.loss(x, target).backward()
    del head.weight.acc_grad
    torch.nn.utils.parametrizations.weight_norm(head)
    head.loss(x, target).backward()
    assert head.parametrizations.weight.original1.grad is not None


def test_gradient_is_that_of_differences():
    """(L(x + h s) - L(x - h s)) / 2h for signs s against <dx, s>, and the same for a word.  The third derivative of log-sum-exp
    along s is the third central moment of the words' slopes under p, at most R^3 / (6 sqrt 3) for slopes of range
    R; x and x +- h s are exact in bf16."""
    from muon_sr_amd import linear_cross_entropy
    g, h = gen(11), 2.0 ** -5
    x = (torch.randint(-16, 17, (6, 64), generator=g, device=DEV) / 16).to(BF16)
    w = (torch.randint(-16, 17, (90, 64), generator=g, device=DEV) / 16).to(BF16)
    target = torch.randint(0, 90, (6,), generator=g, device=DEV)
    (loss, e_loss), (dx, e_dx), (dw, e_dw) = exact(x, w, target, torch.ones(6, device=DEV), "none")
    _, got_dx, got_dw = run(x, w, target, torch.ones(6, device=DEV), "none")
    f = lambda a, b: linear_cross_entropy(a, b, target, reduction="none").double()  # noqa: E731
    for k in range(6):
        s = torch.zeros((6, 64), device=DEV, dtype=BF16)
        s[:, k::6] = torch.randint(0, 2, s[:, k::6].shape, generator=g, device=DEV).to(BF16) * 2 - 1
        diff = (f(x + h * s, w) - f(x - h * s, w)) / (2 * h)
        slopes = s.double() @ w.double().t()
        R = slopes.max(1).values - slopes.min(1).values
        tol = h * h / 6 * R ** 3 / (6 * math.sqrt(3)) + e_loss / h + (e_dx * s.abs()).sum(1)
        assert ((diff - (got_dx.double() * s).sum(1)).abs() <= tol).all()
        # word k along the same signs: its slope in row n is <x[n], s>, those of the others 0
        ws = torch.zeros((90, 64), device=DEV, dtype=BF16)
        ws[k] = s[0]
        diff = (f(x, w + h * ws) - f(x, w - h * ws)).sum() / (2 * h)
        R = (x.double() @ s[0].double()).abs()
        tol = h * h / 6 * (R ** 3).sum() / (6 * math.sqrt(3)) + e_loss.sum() / h + (e_dw[k] * s[0].abs()).sum()
        assert (diff - (got_dw[k].double() * s[0]).sum()).abs() <= tol


@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_the_upstream_gradient_is_not_rounded_with_the_targets(reduction):
    """4096 words that are nearly equally likely: an element of G is g p but for the target's, -g (1 - p), which carries the row.  With
    g = 1 + 2^-8, halfway between two bf16 numbers, it would be off by 2^-8 in every row alike, and so would the gradients be along
    themselves; 1 - p rounds to 1, off by p, which is 2^-12 of the rows on average, and what else is rounded, G's small elements and the
    results, is off to either side: by some 2^-8 / sqrt(elements) along them, less than 2^-16 here.  Twice the former is allowed."""
    g = gen(15)
    x = (torch.randn((512, 256), generator=g, device=DEV) / 64).to(BF16)
    w = torch.randn((4096, 256), generator=g, device=DEV).to(BF16)
    target = torch.randint(0, 4096, (512,), generator=g, device=DEV)
    dloss = torch.full((512,), 1 + 2.0 ** -8, device=DEV)
    _, (dx, _), (dw, _) = exact(x, w, target, dloss, reduction)
    for got, want in zip(run(x, w, target, dloss, reduction)[1:], (dx, dw)):
        along = (got.double() * want).sum() / want.square().sum() - 1
        assert along.abs() <= 2.0 ** -11, along.item()


@pytest.mark.parametrize("size", [30.0, 60.0, 1000.0])
def test_rows_whose_word_is_nearly_sure(size):
    """Logits (exact in fp32) of `size` and more for the target and 20 less for the 63 others: 1 - p is 1.3e-7, 2 u.  In fp32 a row's l has an ulp
    of 32 u and more, but its largest term, the same in both passes, is an exponential of what M leaves of it, off by 2 u by the function; the
    sum by 2 u and the others by what they are; the quotient and its product with that term by 2 u.  8 u bounds the loss and G."""
    k = torch.arange(8, device=DEV)
    x = torch.zeros((8, 8), dtype=BF16, device=DEV)
    x[:, 0] = (size + k / 8 if size < 32 else size + k * size / 128 if size < 64 else 1000 + 4 * k).to(BF16)
    x[:, 1] = -20
    w = torch.zeros((64, 8), dtype=BF16, device=DEV)
    w[:, 0] = 1
    w[1:, 1] = 1
    target = torch.zeros(8, dtype=torch.int64, device=DEV)
    loss, dx, _ = run(x, w, target, torch.ones(8, device=DEV), "none")
    others = 63 * math.exp(-20)
    assert ((loss.double() - math.log1p(others)).abs() <= 8 * U).all(), loss
    assert (dx[:, 0].abs() <= 8 * U).all(), dx[:, 0]                       # the sum of a row of G is 0
    p = others / (1 + others)
    assert ((dx[:, 1].double() - p).abs() <= 2 * H * p).all(), dx[:, 1]


@pytest.mark.parametrize("first", [0.0, -0.0, math.inf, math.nan, 1e-42, 3.4e38, -1.7])
def test_any_first_gradient(first):
    """The first row's upstream gradient, whatever it is, takes part in the others' rows with its significand alone."""
    x, w, target, dloss = make(200, 333, 64, 16, ignored=0.1)
    at = int((target != -100).nonzero()[0])
    dloss[at] = first
    _, got_dx, got_dw = run(x, w, target, dloss, "none")
    others = torch.arange(200, device=DEV) != at
    clean = dloss.clone()
    clean[at] = 0.0
    _, want_dx, want_dw = exact(x, w, target, clean, "none")
    near(got_dx[others], tuple(v[others] for v in want_dx))
    if first == 0.0:
        near(got_dw, want_dw)
        assert not got_dx[at].any()
    elif not math.isfinite(first):
        assert not got_dx[at].isfinite().all()


def test_same_call_same_bits_and_evaluation():
    from muon_sr_amd import linear_cross_entropy
    x, w, target, dloss = make(3000, 8192, 64, 12)
    a = run(x, w, target, dloss, "mean")
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(a, run(x, w, target, dloss, "mean")))
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, target), a[0])
    leaf = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(linear_cross_entropy(leaf, w, target), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.float().sum().backward()


def test_weights_beyond_32_bit_offsets(L):
    """270000 words of 8008: 2.16e9 elements.  The loss, dx, the gradient's last rows and the accumulated ones, whose noise has offsets past
    2^31."""
    import muon_sr_amd as M
    from muon_sr_amd import _lib
    vocab, d, rows = 270000, 8008, 5
    g = gen(13)
    w = torch.randn((vocab, d), generator=g, device=DEV, dtype=BF16).mul_(0.03)
    x = torch.randn((rows, d), generator=g, device=DEV).to(BF16)
    target = torch.tensor([vocab - 1, 3, -100, vocab - 2, 200000], device=DEV)
    dloss = torch.rand(rows, generator=g, device=DEV) + 0.25
    loss, dx, dw = run(x, w, target, dloss, "none")
    S = torch.cat([x.double() @ part.double().t() for part in w.split(30000)], 1)
    eS = 2 * (d + 1) * U * torch.cat([x.double().abs() @ part.double().abs().t() for part in w.split(30000)], 1)
    lse = torch.logsumexp(S, 1)
    el = eS.max(1).values + 2 * (64 + vocab / 64) * U + 8 * U * (lse.abs() + 1) + 2 * U * S.abs().max(1).values
    on = (target != -100).nonzero().flatten()
    near(loss[on], (lse[on] - S[on, target[on]], eS[on, target[on]] + el[on] + U * lse[on].abs()))
    p = torch.exp(S - lse[:, None])
    eG = p * (eS + el[:, None] + 4 * U * ((S - lse[:, None]).abs() + 1) + 2 * U * lse[:, None].abs()) + 2 * U
    G = p.clone()
    G[on, target[on]] -= 1.0
    G, eG = ((torch.where(target != -100, dloss, 0.0).double())[:, None] * v for v in (G, eG))
    eG = eG + H * H * (G.abs() + eG)
    for rows_ in (slice(vocab - 300, vocab), slice(199990, 200010), slice(0, 8)):
        value, terms = G[:, rows_].t() @ x.double(), (eG + 2 * 32 * U * G.abs())[:, rows_].t() @ x.double().abs()
        near(dw[rows_], (value, H * value.abs() + (1 + H) * terms + 1e-30))
    value = torch.zeros((rows, d), dtype=torch.float64, device=DEV)
    terms = torch.zeros_like(value)
    for a in range(0, vocab, 30000):
        part = w[a:a + 30000].double()
        value += G[:, a:a + 30000] @ part
        terms += (eG[:, a:a + 30000] + 2 * (vocab + 16) * U * G[:, a:a + 30000].abs()) @ part.abs()
    near(dx, (value, H * value.abs() + (1 + H) * terms + 1e-30))
    del S, eS, p, G, eG, part
    head = M.SRHead(d, vocab, device="meta")
    head.weight = torch.nn.Parameter(w)
    head.weight.acc_grad = torch.full_like(w, 0.01)
    random.seed(3)
    seed = random.getrandbits(32)
    random.seed(3)
    head.loss(x, target, reduction="none").backward(dloss)
    first = vocab - 40
    noise = torch.empty(40 * d, dtype=torch.int16, device=DEV)
    check(L, L.msr_noise_fill(noise.data_ptr(), noise.numel(), first * d, seed, 0, _lib.noise_mode(), stream()))
    want = torch.full((40, d), 0.01, dtype=BF16, device=DEV)
    check(L, L.msr_sr_accum(want.data_ptr(), dw[first:].contiguous().data_ptr(), 0, want.numel(), 0, 0, _lib.NOISE_INJECT, noise.data_ptr(), stream()))
    assert torch.equal(head.weight.acc_grad[first:], want)


@pytest.mark.parametrize("rows,vocab,d", [(100, 512, 256), (260, 40001, 72), (2047, 3001, 1024), (4096, 8200, 384), (4096, 8200, 2048), (16384, 17001, 64)])
@pytest.mark.parametrize("kept", [1, 5, 14, 32, 100, 128])
def test_few_rows_of_a_padded_batch(rows, vocab, d, kept):
    """The rows that count decide whether G is kept as two numbers (up to 32, 128 where each has its own g), in tiles of every size: their results
    are as near as those of a call of these rows alone.  The other rows' gradients are 0."""
    kept = min(kept, rows - 1)
    x, w, target, dloss = make(rows, vocab, d, rows + kept, ignored=0.0)
    on = torch.sort(torch.randperm(rows, generator=gen(kept), device=DEV)[:kept]).values
    off = torch.ones(rows, dtype=torch.bool, device=DEV)
    off[on] = False
    target[off] = -100
    for reduction in ("mean", "none"):
        if kept > 32 and reduction == "mean":
            continue
        some = dloss[on] if reduction == "none" else dloss
        want = exact(x[on], w, target[on], some, reduction)
        loss, dx, dw = run(x, w, target, dloss, reduction)
        near(loss[on] if reduction == "none" else loss, want[0])
        near(dx[on], want[1])
        near(dw, want[2])
        assert not dx[off].any()


def test_accumulated_gradient_of_few_rows_of_a_padded_batch(L):
    """As the stored one and msr_sr_accum, where G's second numbers are in use in tiles of 256 and of 128."""
    import muon_sr_amd as M
    from muon_sr_amd import _lib
    for rows, vocab, d in ((4096, 8200, 2048), (4096, 8200, 384)):
        x, w, target, dloss = make(rows, vocab, d, 21)
        target[9:] = -100
        head = M.SRHead(d, vocab, device=DEV)
        with torch.no_grad():
            head.weight.copy_(w)
        acc = torch.randn((vocab, d), generator=gen(22), device=DEV).to(BF16)
        head.weight.acc_grad = acc.clone()
        random.seed(3)
        seed = random.getrandbits(32)
        random.seed(3)
        head.loss(x, target).backward(dloss[0])
        dw = run(x, w, target, dloss, "mean")[2]
        check(L, L.msr_sr_accum(acc.data_ptr(), dw.data_ptr(), 0, dw.numel(), seed, 0, _lib.noise_mode(), None, stream()))
        assert torch.equal(head.weight.acc_grad, acc)


def test_hooks_see_the_loss():
    """Forward hooks and pre-hooks of the module run around its loss; a weight that torch.nn.utils' weight_norm or spectral_norm computes
    in a pre-hook is that of the parameters as they are, and its gradient goes to them."""
    import muon_sr_amd as M
    x, _, target, _ = make(50, 100, 64, 23)
    plain = M.SRHead(64, 100, device=DEV)
    seen = []
    plain.register_forward_pre_hook(lambda m, args: (2 * args[0], *args[1:]))
    plain.register_forward_hook(lambda m, args, out: seen.append(out))
    loss = plain.loss(x, target)
    assert torch.equal(loss, M.linear_cross_entropy(2 * x, plain.weight, target)) and seen[0] is loss
    for norm, leaf in ((torch.nn.utils.weight_norm, "weight_g"), (torch.nn.utils.spectral_norm, "weight_orig")):
        head = norm(M.SRHead(64, 100, device=DEV))
        head.eval()                                        # (spectral_norm's estimate stays)
        head.loss(x, target)
        with torch.no_grad():
            getattr(head, leaf).mul_(3)
        loss = head.loss(x, target)
        if norm is torch.nn.utils.weight_norm:
            v = head.weight_v.detach()
            weight = torch._weight_norm(v, head.weight_g.detach(), 0)
        else:
            weight = head.weight_orig.detach()
            weight = weight / torch.dot(head.weight_u, torch.mv(weight, head.weight_v))
        assert torch.equal(loss, M.linear_cross_entropy(x, weight, target))
        loss.backward()
        assert getattr(head, leaf).grad is not None and not hasattr(head.weight, "acc_grad")


@pytest.mark.parametrize("reduction", REDUCTIONS)
@pytest.mark.parametrize("rows,vocab,d", [(300, 1000, 1032), (700, 900, 136), (2047, 3001, 1024), (4096, 8200, 384)])
def test_gradients_are_off_by_their_roundings_alone(rows, vocab, d, reduction):
    """What rounds a gradient, done in 64 bits: G / c to one bf16 number, but for the target's element in dx, whose rest is added exactly, and the
    results.  The kernels' G is nearer to its exact value than 2^-16 of it, so that at most one rounding of 128 falls to the other side, and the norm of
    the errors is that of the roundings within 2 %.  With the target's element rounded in dx too it is 10 to 40 % larger."""
    x, w, target, dloss = make(rows, vocab, d, rows + 24)
    on = target != -100
    X, W, t = x.double()[on], w.double(), target[on]
    g = dloss[on] if reduction == "none" else (dloss[:1] / (int(on.sum()) if reduction == "mean" else 1)).expand(len(t))
    c = 2 * torch.frexp(g[0].double()).mantissa
    at = torch.arange(len(t), device=DEV)
    G = torch.softmax(X @ W.t(), 1)
    G[at, t] -= 1.0
    G *= (g.double() / c)[:, None]
    rounded = G.to(BF16).double()
    own = rounded.clone()
    own[at, t] = G[at, t]
    _, dx, dw = run(x, w, target, dloss, reduction)
    for got, want, model in ((dx[on], G @ W, own @ W), (dw, G.t() @ X, rounded.t() @ X)):
        want, error = c * want, torch.linalg.norm((c * model).to(BF16).double() - c * want)
        assert torch.linalg.norm(got.double() - want) <= 1.02 * error


@pytest.mark.parametrize("rows,vocab", [(200, 9000), (300, 50000), (4096, 9000)])
@pytest.mark.parametrize("size", [8.0, 40.0, 976.0])
def test_nearly_sure_words_of_several_tiles(L, rows, vocab, size):
    """Logits (exact in fp32) of `size` + 25 for the target, which lies in any of several tiles, and of `size` for the others, in more rows than G is
    kept as two numbers for, and tiles of 64 to 256.  1 - p is (vocab - 1) exp(-25), 2 to 12 u, and a row's l has an ulp of 32 u and
    more.  As in the test of a single tile 8 u bounds the loss and the target's element of G: the sum of the word's own tile may lose the tile's
    others, 256 exp(-25) or 0.06 u, and the tiles' sums are joined in 64 bits (in 32 the other tiles, each less than half of 1's ulp, would leave
    nothing: up to 12 u).  The others' elements of G are rounded to 2^-9 of themselves, all to the same side."""
    words = torch.tensor([1, 63, 64, 300, 1111, 4095, 7000, vocab - 1], device=DEV)
    k = torch.arange(rows, device=DEV) % 8
    x = torch.zeros((rows, 16), dtype=BF16, device=DEV)
    x[:, 0] = size
    x[torch.arange(rows, device=DEV), 1 + k] = 25
    w = torch.zeros((vocab, 16), dtype=BF16, device=DEV)
    w[:, 0] = 1
    w[words, 1 + torch.arange(8, device=DEV)] = 1
    assert plan(L, rows, vocab, 16)[0] in ((64, 128) if rows < 300 else (256,))
    loss, dx, _ = run(x, w, words[k], torch.ones(rows, device=DEV), "none")
    one = math.exp(-25)
    others = (vocab - 1) * one
    assert ((loss.double() - math.log1p(others)).abs() <= 8 * U).all(), loss
    assert (dx[:, 0].abs() <= 8 * U + H * others).all(), dx[:, 0]          # the sum of a row of G is 0
    own = torch.zeros((rows, 8), dtype=torch.bool, device=DEV)
    own[torch.arange(rows, device=DEV), k] = True
    G = dx[:, 1:9].double()
    assert ((G[own] + others / (1 + others)).abs() <= 8 * U + H * others).all(), G[own]
    assert ((G[~own] - one / (1 + others)).abs() <= 2 * H * one).all()
