"""Embedding and its gradient against 64-bit evaluations.

Bounds.  With u = 2^-24 and s the type's unit roundoff, a looked-up row is one product, rounded: (s + 2 u) |value|.  A sum
of n rows formed in fp32 is off by at most n u sum|terms|, its product with the scale by 2 u more (the scale itself is rounded to
fp32), and storing adds s |value|: |got - exact| <= s |exact| + 2 (n + 3) u scale sum|terms|."""
import math
import random

import pytest
import torch

from _gpu import DEV, check, need_gpu, stream

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
UNIT = {BF16: 2.0 ** -8, F32: U}


@pytest.fixture(scope="module", autouse=True)
def L():
    return need_gpu()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make(n, vocab, d, dtype, seed, low=0):
    g = gen(seed)
    ids = torch.randint(low, vocab, (n,), generator=g, device=DEV)
    few = torch.rand(n, generator=g, device=DEV) < 0.5
    ids[few] = ids[few] % max(1, vocab // 50)                  # half of the tokens on few words
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    return ids, r(vocab, d), r(n, d)


def want_grad(ids, dy, vocab, scale, padding=None):
    """The gradient, and its bound without the stored value's rounding."""
    keep = (ids >= 0) & (ids < vocab)
    if padding is not None:
        keep &= ids != padding
    ids, dy = ids[keep], dy[keep].double()
    zeros = lambda: torch.zeros((vocab, dy.shape[1]), dtype=torch.float64, device=DEV)  # noqa: E731
    n = torch.zeros(vocab, dtype=torch.float64, device=DEV).index_add_(0, ids, torch.ones(len(ids), dtype=torch.float64, device=DEV))
    value, terms = zeros().index_add_(0, ids, dy) * scale, zeros().index_add_(0, ids, dy.abs()) * abs(scale)
    return value, 2 * (n[:, None] + 3) * U * terms, n


def run(ids, w, dy, scale=1.0, padding=None):
    from muon_sr_amd import embedding
    w = w.detach().requires_grad_(True)
    y = embedding(ids, w, padding_idx=padding, scale=scale)
    return y.detach(), torch.autograd.grad(y, w, dy)[0]


def compare(ids, w, dy, scale=1.0, padding=None):
    y, dw = run(ids, w, dy, scale, padding)
    vocab, unit = w.shape[0], UNIT[w.dtype]
    there = (ids >= 0) & (ids < vocab)
    want = torch.where(there[:, None], w[ids.clamp(0, vocab - 1).long()].double() * scale, 0.0)
    assert y.dtype == w.dtype and ((y.double() - want).abs() <= (unit + 2 * U) * want.abs()).all()
    if scale == 1.0:
        assert torch.equal(y.double(), want)
    value, bound, n = want_grad(ids.long(), dy, vocab, scale, padding)
    assert dw.dtype == w.dtype and ((dw.double() - value).abs() <= unit * value.abs() + bound).all()
    assert not dw[n == 0].any()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n,vocab,d", [(1, 1, 1), (1, 5, 8), (61, 512, 256), (33, 7, 3), (64, 64, 384), (1000, 3, 129), (1025, 5000, 520),
                                       (5000, 130000, 16), (16384, 1000, 40), (16385, 512, 24), (40001, 70000, 9), (70000, 300, 8), (3001, 4, 1100)])
def test_against_64_bits(n, vocab, d, dtype):
    compare(*make(n, vocab, d, dtype, n + vocab))
    ids, w, dy = make(n, vocab, d, dtype, n + vocab + 1, low=-1)           # some without a word
    ids[::7] = vocab + 3
    ids[::11] = (1 << 40) + 1 if n > 50 else ids[::11]
    compare(ids, w, dy, scale=math.sqrt(d))
    compare(ids, w, dy, scale=0.37, padding=vocab // 3)
    compare(torch.where((ids < 0) | (ids > vocab), -1, ids).int(), w, dy)


def test_words_that_span_many_chunks():
    """One word for all tokens; a few; and runs whose borders fall on those of the 16- and 32-token chunks and one beside (more than
    512 tokens, which are sorted; as many words as tokens for chunks of 32)."""
    g = gen(2)
    for n in (31, 32, 33, 64, 65, 4096, 20000, 50001):
        dy = torch.randn((n, 72), generator=g, device=DEV).to(BF16)
        w = torch.randn((12, 72), generator=g, device=DEV).to(BF16)
        compare(torch.full((n,), 4, device=DEV), w, dy)
        compare((torch.arange(n, device=DEV) * 3 // n) * 5, w, dy)
    for lengths in ([32, 32, 64, 31, 1, 33], [1, 31, 32, 96, 2], [63, 65, 64, 5], [16, 16, 16, 16, 128], [15, 1, 17, 15, 16, 48]):
        for more in (0, 512, 528):
            lengths_ = lengths + [more]
            ids = torch.repeat_interleave(torch.arange(len(lengths_), device=DEV), torch.tensor(lengths_, device=DEV))
            ids = ids[torch.randperm(len(ids), generator=g, device=DEV)]
            for vocab in (9, 900):
                compare(ids, torch.randn((vocab, 72), generator=g, device=DEV).to(BF16), torch.randn((len(ids), 72), generator=g, device=DEV).to(BF16))


def test_nothing_to_look_up():
    w = torch.randn((7, 16), device=DEV).to(BF16)
    y, dw = run(torch.zeros((0, 3), dtype=torch.int64, device=DEV), w, torch.zeros((0, 3, 16), dtype=BF16, device=DEV))
    assert y.shape == (0, 3, 16) and dw.shape == w.shape and not dw.any()
    y, dw = run(torch.full((5,), -1, device=DEV), w, torch.ones((5, 16), dtype=BF16, device=DEV))
    assert not y.any() and not dw.any()
    y, dw = run(torch.tensor(3, device=DEV), w, torch.ones(16, dtype=BF16, device=DEV))
    assert torch.equal(y, w[3]) and torch.equal(dw.sum(0), torch.ones(16, dtype=BF16, device=DEV))
    y, dw = run(torch.zeros(4, dtype=torch.int64, device=DEV), w[:, :0].contiguous(), torch.zeros((4, 0), dtype=BF16, device=DEV))
    assert y.shape == (4, 0) and dw.shape == (7, 0)


def test_rows_that_no_token_wants_reach_nothing():
    """NaN in the gradient of tokens without a word, or of padding, and in the rows of other words."""
    ids, w, dy = make(500, 90, 48, BF16, 3)
    ids[::5], ids[::6] = -1, 17
    want = run(ids, w, dy, padding=17)[1]
    dirty = dy.clone()
    dirty[(ids < 0) | (ids == 17)] = math.nan
    assert torch.equal(run(ids, w, dirty, padding=17)[1], want) and not want[17].any()
    unused = torch.ones(90, dtype=torch.bool, device=DEV)
    unused[ids.clamp(min=0)[ids >= 0]] = False
    spoilt = torch.where(unused[:, None], math.nan, w)
    assert torch.equal(run(ids, spoilt, dy)[0], run(ids, w, dy)[0])


def test_strides_and_padding_from_the_end():
    from muon_sr_amd import embedding
    ids, w, dy = make(120, 50, 24, BF16, 4)
    want = run(ids, w, dy, padding=49)
    wide = torch.zeros((120, 64), dtype=BF16, device=DEV)
    wide[:, 5:29] = dy
    cases = [wide[:, 5:29], dy.t().contiguous().t()]
    for v in cases:
        assert torch.equal(run(ids, w, v, padding=-1)[1], want[1])
    assert torch.equal(run(ids.view(10, 12), w, dy.view(10, 12, 24), padding=49)[1], want[1])
    turned = ids.view(10, 12).t()
    assert torch.equal(embedding(turned, w), w[turned])
    one = torch.ones((1, 24), dtype=BF16, device=DEV).expand(120, 24)
    assert torch.equal(run(ids, w, one)[1], run(ids, w, one.contiguous())[1])


@pytest.mark.parametrize("noise", ["philox8", "triton"])
@pytest.mark.parametrize("n,vocab,d", [(61, 512, 256), (700, 90, 13), (20000, 333, 72), (1, 4, 8), (5000, 130000, 16), (3001, 4, 1100)])
def test_accumulated(L, n, vocab, d, noise):
    """Bit for bit the stored gradient and msr_sr_accum, for the words that tokens hit; the others are untouched."""
    import muon_sr_amd as M
    from muon_sr_amd import _lib
    layer = M.SREmbedding(vocab, d, padding_idx=2, scale=1.5, device=DEV)
    was = M.get_sr_noise()
    M.set_sr_noise(noise)
    try:
        acc = None
        for micro in range(3):
            ids, w, dy = make(n, vocab, d, BF16, micro, low=-1)
            with torch.no_grad():
                layer.weight.copy_(w)
            random.seed(micro)
            seed = random.getrandbits(32)
            random.seed(micro)
            layer(ids).backward(dy)
            dw = run(ids, w, dy, 1.5, 2)[1]
            want = torch.empty_like(dw) if acc is None else acc.clone()
            check(L, L.msr_sr_accum(want.data_ptr(), dw.data_ptr(), 0, dw.numel(), seed, int(acc is None), _lib.noise_mode(), None, stream()))
            hit = torch.zeros(vocab, dtype=torch.bool, device=DEV)
            hit[ids[(ids >= 0) & (ids != 2)]] = True
            got = layer.weight.acc_grad
            assert layer.weight.grad is None and torch.equal(got[hit], want[hit])
            assert torch.equal(got[~hit], torch.zeros_like(got[~hit]) if acc is None else acc[~hit])
            acc = got.clone()
    finally:
        M.set_sr_noise(was)


@pytest.mark.parametrize("n,vocab,d", [(3000, 3500, 512), (3000, 20000, 512), (5000, 700, 520)])
def test_accumulated_sums_have_the_order_of_the_stored_ones(L, n, vocab, d):
    """A word whose partial sums are thousands of times as large as their end, so that another order would give other bits: accumulating into a
    buffer that is there gives what the stored gradient and msr_sr_accum give."""
    from muon_sr_amd import _lib, embedding_grad_sr_accum
    g = gen(9)
    ids = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    ids[torch.rand(n, generator=g, device=DEV) < 0.5] = 3
    dy = torch.randn((n, d), generator=g, device=DEV).to(BF16)
    same = (ids == 3).nonzero().flatten()
    m = len(same) // 3
    dy[same[:m]] *= 4096
    dy[same[m:2 * m]] = -dy[same[:m]]
    w = torch.nn.Parameter(torch.zeros((vocab, d), dtype=BF16, device=DEV))
    dw = run(ids, w, dy)[1]
    want = torch.randn((vocab, d), generator=g, device=DEV).to(BF16)
    w.acc_grad = want.clone()
    embedding_grad_sr_accum(w, ids, dy, seed=5)
    check(L, L.msr_sr_accum(want.data_ptr(), dw.data_ptr(), 0, dw.numel(), 5, 0, _lib.noise_mode(), None, stream()))
    hit = torch.zeros(vocab, dtype=torch.bool, device=DEV)
    hit[ids] = True
    assert torch.equal(w.acc_grad[hit], want[hit])


def test_refusals_and_other_weights():
    import muon_sr_amd as M
    ids, w, dy = make(30, 40, 16, BF16, 5)
    layer = M.SREmbedding(40, 16, device=DEV)
    for bad in (torch.zeros((40, 16), device=DEV), torch.zeros((16, 40), dtype=BF16, device=DEV).t(), None):
        layer.weight.acc_grad = bad
        with pytest.raises(ValueError, match="acc_grad"):
            layer(ids).backward(dy)
    del layer.weight.acc_grad
    wide = M.SREmbedding(40, 16, device=DEV, dtype=F32)
    wide(ids).backward(dy.float())
    assert wide.weight.grad.dtype == F32 and not hasattr(wide.weight, "acc_grad")
    torch.nn.utils.parametrizations.weight_norm(layer)
    layer(ids).backward(dy)
    assert layer.parametrizations.weight.original1.grad is not None
    for call in (lambda: M.embedding(ids, w, padding_idx=40), lambda: M.embedding(ids.float(), w), lambda: M.embedding(ids, w.half()),
                 lambda: M.embedding(ids, w.t()), lambda: M.embedding_grad_sr_accum(w, ids, dy[1:]),
                 lambda: M.embedding_grad_sr_accum(w.float(), ids, dy.float()), lambda: M.embedding(ids.cpu(), w)):
        with pytest.raises(ValueError):
            call()


def test_gradient_is_that_of_differences():
    """The sum of y c is linear in the weight: its difference along any direction is <dw, direction> but for roundings.  With
    whole numbers (up to 5 x 3 x 90 terms) there are none."""
    from muon_sr_amd import embedding
    g = gen(6)
    ids = torch.randint(-1, 11, (90,), generator=g, device=DEV)
    whole = lambda *s: torch.randint(-3, 4, s, generator=g, device=DEV).float()  # noqa: E731
    w, dy, step = whole(10, 24), whole(90, 24), whole(10, 24)
    f = lambda v: (embedding(ids, v) * dy).sum()  # noqa: E731
    dw = run(ids, w, dy)[1]
    assert torch.equal(f(w + step) - f(w - step), 2 * (dw * step).sum())


def test_same_call_same_bits():
    ids, w, dy = make(50000, 700, 136, BF16, 7)
    a = run(ids, w, dy)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(a, run(ids, w, dy)))


def test_weights_beyond_32_bit_offsets(L):
    """270000 words of 8008: 2.16e9 elements, with tokens on the last ones; the accumulator's noise has offsets past 2^31."""
    import muon_sr_amd as M
    from muon_sr_amd import _lib
    vocab, d = 270000, 8008
    g = gen(8)
    w = torch.nn.Parameter(torch.randn((vocab, d), generator=g, device=DEV, dtype=BF16))
    for n in (50, 1200):
        ids = torch.cat([torch.randint(vocab - 30, vocab, (n // 2,), generator=g, device=DEV), torch.randint(0, vocab, (n // 2,), generator=g, device=DEV)])
        dy = torch.randn((n, d), generator=g, device=DEV).to(BF16)
        y = M.embedding(ids, w)
        assert torch.equal(y, w[ids])
        dw, = torch.autograd.grad(y, w, dy)
        first = vocab - 30
        late = ids >= first
        value, bound, count = want_grad(torch.where(late, ids - first, -1), dy, 30, 1.0)
        assert ((dw[first:].double() - value).abs() <= UNIT[BF16] * value.abs() + bound).all()
        assert int((dw != 0).any(1).sum()) == len(ids.unique())
        w.acc_grad = torch.full_like(w, 0.5)
        M.embedding_grad_sr_accum(w, ids, dy, seed=77)
        noise = torch.empty(30 * d, dtype=torch.int16, device=DEV)
        check(L, L.msr_noise_fill(noise.data_ptr(), noise.numel(), first * d, 77, 0, _lib.noise_mode(), stream()))
        want = torch.full((30, d), 0.5, dtype=BF16, device=DEV)
        check(L, L.msr_sr_accum(want.data_ptr(), dw[first:].contiguous().data_ptr(), 0, want.numel(), 0, 0, _lib.NOISE_INJECT, noise.data_ptr(), stream()))
        assert torch.equal(w.acc_grad[first:], torch.where((count > 0)[:, None], want, 0.5))
        assert torch.equal((w.acc_grad != 0.5).any(1).nonzero().flatten(), ids.unique())
        del w.acc_grad, dw


def test_from_pretrained():
    """The module of given embeddings looks them up, and accumulates where it is not frozen."""
    import muon_sr_amd as M
    ids, w, dy = make(700, 90, 24, BF16, 10)
    assert torch.equal(M.SREmbedding.from_pretrained(w, scale=2.0)(ids), run(ids, w, dy, 2.0)[0])
    layer = M.SREmbedding.from_pretrained(w, freeze=False, padding_idx=3)
    random.seed(1)
    layer(ids).backward(dy)
    want = torch.nn.Parameter(w)
    random.seed(1)
    M.embedding_grad_sr_accum(want, ids, dy, padding_idx=3)
    assert layer.weight.grad is None and torch.equal(layer.weight.acc_grad, want.acc_grad)
