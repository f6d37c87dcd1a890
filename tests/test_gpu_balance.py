"""The router's balance loss against its definition in 64 bits.

Bounds, with u = 2^-24.  exp of an argument a costs 4 u (|a| + 1) (the difference, its product with log2 e, that constant, the
function); the sum of E of them is off by E u more, and its reciprocal within 2 u, so a probability is off by ep = p (4 u (|x - max| + 1) + 2 (E + 8) u), and from the
stored log-sum-exp l by u (|l| + 1) p more.  The mean over n tokens adds (n + 8) u, the loss's stored value u.
dlogits = up p (u_e - sum_j u_j p_j): up (ep |.| + p (sum u_j ep_j + (E + 4) u sum u_j p_j)) + 4 u |value|, and the
stored value's rounding."""
import math

import numpy as np
import pytest
import torch

from _gpu import DEV, need_gpu

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
UNIT = {BF16: 2.0 ** -8, F32: U}


@pytest.fixture(scope="module", autouse=True)
def L():
    return need_gpu()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make(tokens, experts, k, dtype, seed, dropped=0.1, masked=0.2):
    g = gen(seed)
    logits = (2 * torch.randn((tokens, experts), generator=g, device=DEV) + torch.randn(experts, generator=g, device=DEV)).to(dtype)
    ids = torch.randint(0, experts, (tokens, k), generator=g, device=DEV)
    ids[torch.rand((tokens, k), generator=g, device=DEV) < dropped] = -1
    mask = torch.rand(tokens, generator=g, device=DEV) >= masked if masked else None
    return logits, ids, mask, torch.tensor(0.73, device=DEV)


def exact(logits, ids, mask, up):
    tokens, E = logits.shape
    on = torch.ones(tokens, dtype=torch.bool, device=DEV) if mask is None else mask
    flat = ids[on].cpu().numpy().reshape(-1)
    counts = np.bincount(flat[(flat >= 0) & (flat < E)], minlength=E)
    n = max(1, int(on.sum()))
    slope = torch.from_numpy(counts * (E / (n * ids.shape[1] * n))).to(DEV)
    x = torch.where(on[:, None], logits.double(), 0.0)
    top = x.max(1, keepdim=True).values
    some = on[:, None] & (top > -math.inf)
    x, top = torch.where(some, x, 0.0), torch.where(some, top, 0.0)
    lse = torch.logsumexp(x, 1, keepdim=True)
    p = torch.where(some, torch.exp(x - lse), 0.0)
    far = torch.where(p > 0, (x - top).abs(), 0.0)
    ep = p * (4 * U * (far + 1) + 2 * (E + 8) * U + U * (lse.abs() + 1) + 4 * U * (far + lse.abs()))
    loss = (p.sum(0) * slope).sum()
    e_loss = (ep.sum(0) * slope).sum() + (n + 16) * U * loss
    dot = (p * slope).sum(1, keepdim=True)
    d = up.double() * p * (slope - dot)
    ed = up.double() * (ep * (slope - dot).abs() + p * ((ep * slope).sum(1, keepdim=True) + (E + 4) * U * dot + 4 * U * slope)) + 4 * U * d.abs()
    return counts, (loss, e_loss), (d, ed)


def run(logits, ids, mask, up):
    from muon_sr_amd import balance_loss
    leaf = logits.detach().requires_grad_(True)
    loss, counts = balance_loss(leaf, ids, mask)
    assert loss.dtype == F32 and counts.dtype == torch.int32 and not counts.requires_grad
    return loss.detach(), counts, torch.autograd.grad(loss, leaf, up)[0]


def compare(logits, ids, mask, up):
    loss, counts, d = run(logits, ids, mask, up)
    want, (value, bound), (slope, e) = exact(logits, ids, mask, up)
    assert np.array_equal(counts.cpu().numpy(), want)
    assert abs(loss.item() - value.item()) <= bound.item() + 2 * U * value.item()
    assert d.dtype == logits.dtype and ((d.double() - slope).abs() <= e + UNIT[d.dtype] * (slope.abs() + e) + 2.0 ** -126).all()
    return d


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 2, 2), (7, 8, 2), (65, 9, 1), (1000, 16, 3), (333, 17, 2), (64, 33, 4), (8192, 64, 2),
                                              (301, 65, 2), (5000, 128, 8), (77, 200, 6), (2050, 257, 2), (513, 512, 4), (260, 1000, 70),
                                              (1025, 1024, 8), (130001, 12, 2)])
def test_against_64_bits(tokens, experts, k, dtype):
    compare(*make(tokens, experts, k, dtype, tokens + experts))
    compare(*make(tokens, experts, k, dtype, tokens + experts + 1, dropped=0.0, masked=0.0))


def test_masked_tokens_reach_nothing():
    logits, ids, mask, up = make(400, 24, 2, F32, 1)
    want = run(logits, ids, mask, up)
    dirty, wrong = logits.clone(), ids.clone()
    dirty[~mask], wrong[~mask] = math.nan, 5
    got = run(dirty, wrong, mask, up)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not got[2][~mask].any()
    loss, counts, d = run(dirty, ids, torch.zeros_like(mask), up)
    assert loss.item() == 0.0 and not counts.any() and not d.any()


def test_no_tokens():
    loss, counts, d = run(torch.zeros((0, 6), device=DEV), torch.zeros((0, 2), dtype=torch.int64, device=DEV), None, torch.ones((), device=DEV))
    assert loss.item() == 0.0 and not counts.any() and d.shape == (0, 6)


def test_infinite_and_far_logits():
    """Experts at -inf or the type's lowest value have probability 0; a token of nothing else counts with 0; NaN stays in its row."""
    for dtype in (BF16, F32):
        logits, ids, _, up = make(300, 40, 2, dtype, 2, masked=0.0)
        logits[::3, 5:9] = -math.inf
        logits[1::3, 7] = torch.finfo(dtype).min
        logits[10], logits[200] = -math.inf, -math.inf
        logits[20, 3] = torch.finfo(dtype).max
        d = compare(logits, ids, None, up)
        assert not d[::3, 5:9].any() and not d[1::3, 7].any() and not d[10].any()
        logits[33, 2] = math.nan
        loss, counts, got = run(logits, ids, None, up)
        others = torch.arange(300, device=DEV) != 33
        assert loss.isnan() and got[33].isnan().any() and torch.equal(got[others], d[others])


def test_even_load_is_one():
    logits = torch.zeros((640, 32), device=DEV)
    ids = (torch.arange(1280, device=DEV) % 32).view(640, 2)
    loss, counts, d = run(logits, ids, None, torch.ones((), device=DEV))
    assert abs(loss.item() - 1.0) <= 32 * U and torch.equal(counts, torch.full((32,), 40, dtype=torch.int32, device=DEV))


def test_strides_types_and_refusals():
    from muon_sr_amd import balance_loss
    logits, ids, mask, up = make(120, 20, 2, F32, 3)
    want = run(logits, ids, mask, up)
    wide = torch.zeros((120, 64), device=DEV)
    wide[:, 7:27] = logits
    both = torch.stack([mask, mask], 1)[:, 0]
    for case in ((wide[:, 7:27], ids, mask, up), (logits.t().contiguous().t(), ids.t().contiguous().t(), both, up), (logits, ids.int(), mask, up)):
        assert all(torch.equal(a, b) for a, b in zip(run(*case), want))
    huge = ids.clone()
    huge[::9, 0] = (1 << 40) + 3
    compare(logits, huge, mask, up)
    for bad in (lambda: balance_loss(logits, ids[:5]), lambda: balance_loss(logits.half(), ids), lambda: balance_loss(logits, ids.float()),
                lambda: balance_loss(logits, ids, mask.int()), lambda: balance_loss(logits, ids, mask[:4]), lambda: balance_loss(logits, ids.cpu()),
                lambda: balance_loss(torch.zeros((3, 1025), device=DEV), torch.zeros((3, 1), dtype=torch.int64, device=DEV))):
        with pytest.raises(ValueError):
            bad()


def test_gradient_is_that_of_differences():
    """The loss is sum_e u_e sum_t p: along v its third derivative is at most E sum_t |v_t|^3 max u; the loss itself is exact to
    (E + 16) 2^-22, which the step divides."""
    from muon_sr_amd import balance_loss
    logits, ids, mask, _ = make(40, 24, 2, F32, 4)
    d = run(logits, ids, mask, torch.ones((), device=DEV))[2].double()
    u = (balance_loss(logits, ids, mask)[1].double() * 24 / (2 * mask.sum() ** 2)).max()
    h = 2.0 ** -5
    for k in range(5):
        v = torch.randint(-1, 2, (40, 24), generator=gen(30 + k), device=DEV).float()
        hi, lo = logits + h * v, logits - h * v
        diff = (balance_loss(hi, ids, mask)[0].double() - balance_loss(lo, ids, mask)[0].double()) / (2 * h)
        step = (hi.double() - lo.double()) / (2 * h)
        tol = h * h / 6 * 24 * (mask * v.norm(dim=1) ** 3).sum() * u + (24 + 16) * 2.0 ** -22 * 2 / h
        assert abs(diff - (d * step).sum()) <= tol


def test_same_call_same_bits():
    case = make(50000, 100, 4, BF16, 5)
    a = run(*case)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(a, run(*case)))


@pytest.mark.parametrize("tokens,experts", [(8192, 64), (2050, 257), (513, 1000)])
@pytest.mark.parametrize("offset", [0.0, 1000.0, -10000.0])
def test_logits_far_from_zero_and_an_even_load(tokens, experts, offset):
    """Every expert has nearly the same load, so that u[e] - sum_j u[j] p[j] is small beside u: an error that all p of a token have in common
    remains in dlogits as that error times u p.  p is formed from a maximum and a sum, whatever size the logits have: exp costs 4 u (|x - max| + 1), the
    sum has at most 16 additions in a lane and 6 of a wave's after one another, its reciprocal and the product with it 3 u.  The log of the sum
    added to the maximum would be off by up to u |offset|."""
    g = gen(40 + tokens)
    logits = offset + torch.randn((tokens, experts), generator=g, device=DEV)
    ids = (torch.arange(2 * tokens, device=DEV) % experts).view(tokens, 2)
    ids[:tokens // 100, 0] = 3
    up = torch.tensor(0.73, device=DEV)
    _, counts, d = run(logits, ids, None, up)
    x = logits.double()
    p = torch.softmax(x, 1)
    ep = p * (4 * U * ((x.amax(1, keepdim=True) - x) + 1) + (16 + 6 + 4) * U)
    slope = counts.double() * experts / (2 * tokens * tokens)
    dot, edot = (p * slope).sum(1, keepdim=True), ((ep + 26 * U * p) * slope).sum(1, keepdim=True)
    want = up.double() * p * (slope - dot)
    bound = up.double() * (ep * (slope - dot).abs() + p * (edot + 4 * U * slope)) + 4 * U * want.abs()
    assert ((d.double() - want).abs() <= bound).all()


def test_more_than_2_31_elements():
    """2.2 million tokens of 1024 experts: the counts are those of numpy, the last tokens' gradients those of the formula."""
    tokens, experts = 2200000, 1024
    g = gen(50)
    logits = torch.randn((tokens, experts), generator=g, device=DEV, dtype=BF16)
    ids = torch.randint(0, experts, (tokens, 1), generator=g, device=DEV)
    loss, counts, d = run(logits, ids, None, torch.ones((), device=DEV))
    assert torch.equal(counts.long(), torch.bincount(ids.flatten(), minlength=experts))
    slope = counts.double() * experts / (float(tokens) * tokens)
    total = sum((torch.softmax(part.double(), 1).sum(0) * slope).sum().item() for part in logits.split(50000))
    # sums of tokens / 4096 probabilities in a lane, then of 16 waves' and of 256 work-groups'; a probability is off by 100 u of itself at most:
    # 4 u (|x - max| + 1) for logits that are up to 11 apart, and 40 u for its sum and quotient
    assert abs(loss.item() - total) <= (tokens / 4096 + 16 + 256 + 100) * U * total
    p = torch.softmax(logits[-500:].double(), 1)
    dot = (p * slope).sum(1, keepdim=True)
    want = p * (slope - dot)
    far = logits[-500:].double().amax(1, keepdim=True) - logits[-500:].double()
    ep = p * (4 * U * (far + 1) + 40 * U)
    bound = ep * (slope - dot).abs() + p * ((ep * slope).sum(1, keepdim=True) + 40 * U * dot + 4 * U * slope)
    assert ((d[-500:].double() - want).abs() <= bound + UNIT[BF16] * (want.abs() + bound) + 2.0 ** -126).all()
