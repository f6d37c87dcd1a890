"""Tokens sorted by expert and back, against plain 64-bit evaluations.

Bounds.  With u = 2^-24 (fp32) and s the type's unit roundoff (2^-8 for bf16: 8 significant bits; u for fp32), a sum of n
products formed in fp32 differs from the exact one by at most (n + 1) u sum|terms|, and storing adds
s |value|: |got - exact| <= s |exact| + 2 (n + 1) u sum|terms|  (the factor 2 covers the stored value's own
error).  Copies are compared bit for bit, orders exactly."""
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


def plain_order(ids, E):
    flat = ids.reshape(-1)
    lists = [np.nonzero(flat == e)[0] for e in range(E)]
    offsets = np.concatenate([[0], np.cumsum([len(x) for x in lists])])
    kept = np.concatenate(lists)
    source = np.full(flat.size, -1)
    source[:kept.size] = kept
    position = np.full(flat.size, -1)
    position[kept] = np.arange(kept.size)
    return offsets, position.reshape(ids.shape), source


def check_order(ids, E, dtype=torch.int64):
    from muon_sr_amd import order_tokens
    order = order_tokens(torch.from_numpy(ids).to(dtype).to(DEV), E)
    for got, want in zip(order, plain_order(ids, E)):
        assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), want)
    return order


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=["int32", "int64"])
@pytest.mark.parametrize("tokens,k,E", [(1, 1, 1), (7, 2, 8), (64, 1, 3), (65, 3, 64), (1000, 2, 65), (1024, 2, 255),
                                        (2049, 1, 256), (683, 3, 1023), (5000, 8, 1024), (70001, 4, 130),
                                        (300000, 2, 7), (40000, 2, 1000), (66000, 8, 500)])
def test_order(tokens, k, E, dtype):
    rng = np.random.default_rng(tokens + E)
    check_order(rng.integers(0, E, (tokens, k)), E, dtype)
    # uneven, with slots that have no expert: negative ids and too large ones
    skew = np.minimum(rng.geometric(0.3, (tokens, k)) - 2, E + 3)
    check_order(skew, E, dtype)


def test_order_extremes():
    check_order(np.zeros((0, 2), dtype=np.int64), 5)
    check_order(np.full((3001, 2), 4), 5)
    check_order(np.full((3001, 2), -1), 5)
    check_order(np.tile(np.arange(128)[::-1], (40, 1)), 128)
    ids = np.random.default_rng(0).integers(0, 16, (900, 3))
    ids[::7, 1] = 1 << 40                       # out of range in its high word only
    ids[::5, 0] = -(1 << 33) + 3
    check_order(ids, 16)


def test_no_tokens_and_no_width():
    from muon_sr_amd import combine_tokens, dispatch_tokens, order_tokens
    order = order_tokens(torch.zeros((0, 2), dtype=torch.int64, device=DEV), 3)
    x, w = torch.zeros((0, 16), device=DEV, requires_grad=True), torch.zeros((0, 2), device=DEV, requires_grad=True)
    y = combine_tokens(dispatch_tokens(x, order), w, order)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros((0, 16), device=DEV))
    assert y.shape == dx.shape == (0, 16) and dw.shape == (0, 2)
    s = make(5, 2, 3, 0, BF16, F32, 1)
    moved, y, dx, dr, dw = all_passes(s)
    assert moved.shape == dr.shape == (10, 0) and y.shape == dx.shape == (5, 0) and dw.shape == (5, 2) and not dw.any()


def test_order_of_strided_ids():
    from muon_sr_amd import order_tokens
    ids = torch.randint(0, 9, (100, 12), generator=gen(1), device=DEV)
    for got, want in zip(order_tokens(ids[:, 3:5], 9), plain_order(ids[:, 3:5].cpu().numpy(), 9)):
        assert np.array_equal(got.cpu().numpy(), want)


def make(tokens, k, E, d, dtype, wdtype, seed, dropped=0.2):
    from muon_sr_amd import order_tokens
    g = gen(seed)
    ids = torch.randint(0, E, (tokens, k), generator=g, device=DEV)
    ids[torch.rand((tokens, k), generator=g, device=DEV) < dropped] = -1
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    return dict(order=order_tokens(ids, E), x=r(tokens, d).to(dtype), rows=r(tokens * k, d).to(dtype),
                w=torch.rand((tokens, k), generator=g, device=DEV).to(wdtype), dy=r(tokens, d).to(dtype),
                drows=r(tokens * k, d).to(dtype))


def near(got, exact, terms, n):
    """terms: sum of the terms' magnitudes."""
    got = got.double()
    bound = UNIT[BF16 if terms["dtype"] == BF16 else F32] * exact.abs() + 2 * (n + 1) * U * terms["sum"]
    assert bool(torch.isfinite(got).all()) and bool(((got - exact).abs() <= bound).all())


def all_passes(s, x=None, rows=None, dy=None, drows=None):
    from muon_sr_amd import combine_tokens, dispatch_tokens
    x = (s["x"] if x is None else x).detach().requires_grad_(True)
    rows = (s["rows"] if rows is None else rows).detach().requires_grad_(True)
    w = s["w"].detach().requires_grad_(True)
    moved = dispatch_tokens(x, s["order"])
    y = combine_tokens(rows, w, s["order"])
    grads = torch.autograd.grad((moved, y), (x, rows, w), (s["drows"] if drows is None else drows, s["dy"] if dy is None else dy))
    return (moved, y, *grads)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("wdtype", [BF16, F32], ids=["wbf16", "wfp32"])
@pytest.mark.parametrize("tokens,k,E,d", [(1, 1, 1, 1), (1, 2, 4, 8), (7, 2, 8, 384), (33, 3, 5, 100), (130, 1, 64, 513),
                                          (64, 8, 16, 1400), (513, 5, 40, 2048), (5, 2, 3, 8200), (9000, 2, 16, 48),
                                          (70, 11, 13, 264), (40, 4, 6, 4098),
                                          (21, 70, 90, 136), (5, 129, 40, 600)])
def test_passes(tokens, k, E, d, dtype, wdtype):
    s = make(tokens, k, E, d, dtype, wdtype, tokens + d)
    o = s["order"]
    moved, y, dx, dr, dw = all_passes(s)
    there = (o.position >= 0).unsqueeze(2)
    at = o.position.clamp(min=0).long()
    token = o.source.clamp(min=0).long() // k
    held = (o.source >= 0).unsqueeze(1)
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    # copies
    assert torch.equal(moved, torch.where(held, s["x"][token], torch.zeros_like(moved)))
    # y
    w, r, g = s["w"].double(), s["rows"].double(), s["dy"].double()
    picked = torch.where(there, r[at], zero)
    terms = picked * w.unsqueeze(2)
    near(y, terms.sum(1), dict(dtype=dtype, sum=terms.abs().sum(1)), k)
    # dx
    back = torch.where(there, s["drows"].double()[at], zero)
    near(dx, back.sum(1), dict(dtype=dtype, sum=back.abs().sum(1)), k)
    # dr: one product
    exact = torch.where(held, g[token] * w.flatten()[o.source.clamp(min=0).long()].unsqueeze(1), zero)
    near(dr, exact, dict(dtype=dtype, sum=exact.abs()), 0)
    # dw: d products
    terms = picked * g.unsqueeze(1)
    near(dw, terms.sum(2), dict(dtype=wdtype, sum=terms.abs().sum(2)), d)
    assert not dw[o.position < 0].any()
    # the same bits again
    assert all(torch.equal(a, b) for a, b in zip((moved, y, dx, dr, dw), all_passes(s)))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("tokens,k,E,d", [(1, 2, 3, 2056), (5, 70, 9, 4104), (3, 3, 5, 9000), (6, 2, 5, 9003), (4099, 1, 4, 270),
                                          (20011, 2, 4, 1032)])
def test_rows_of_several_pieces(tokens, k, E, d, dtype):
    """Rows that several waves share, more of them than one round of the launch, and slots beyond a wave's lanes."""
    test_passes(tokens, k, E, d, dtype, F32)


def test_strides_and_alignment():
    """x and dy with row strides, unaligned starts, transposed: the same bits as contiguous ones."""
    s = make(77, 2, 6, 96, BF16, F32, 1)
    want = all_passes(s)
    wide = torch.zeros(77, 200, dtype=BF16, device=DEV)
    for first in (0, 8, 3):
        x, dy = wide[:, first:first + 96], wide.clone()[:, 104 - first:200 - first]
        x.copy_(s["x"])
        dy.copy_(s["dy"])
        assert all(torch.equal(a, b) for a, b in zip(want, all_passes(s, x=x, dy=dy)))
    turned = s["rows"].t().contiguous().t()
    assert all(torch.equal(a, b) for a, b in zip(want, all_passes(s, rows=turned, drows=s["drows"].t().contiguous().t())))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_rows_without_a_slot_are_not_read(dtype):
    """NaN and infinity in rows without a slot reach nothing; those rows get zeros."""
    s = make(300, 3, 7, 128, dtype, F32, 2, dropped=0.5)
    n = int(s["order"].offsets[-1])
    clean = all_passes(s)
    s["rows"][n:] = float("nan")
    s["drows"][n:] = float("inf")
    for a, b in zip(clean, all_passes(s)):
        assert torch.equal(a, b)
    assert not clean[0][n:].any() and not clean[3][n:].any()
    # a token all of whose slots are dropped
    alone = (s["order"].position < 0).all(1)
    assert bool(alone.any()) and not clean[1][alone].any() and not clean[2][alone].any()


def test_expanded_gradients():
    s = make(20, 2, 3, 64, BF16, F32, 3)
    ones = torch.ones((), dtype=BF16, device=DEV)
    a = all_passes(s, dy=ones.expand(20, 64), drows=ones.expand(40, 64))
    b = all_passes(s, dy=torch.ones(20, 64, dtype=BF16, device=DEV), drows=torch.ones(40, 64, dtype=BF16, device=DEV))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradients_against_differences():
    """combine is linear in the rows and in the weights, dispatch in x: differences of any step are the
    derivatives, up to the fp32 rounding of the two sums (k + 1 terms of order 1 at step 1: 1e-5 holds ten times that)."""
    from muon_sr_amd import combine_tokens, dispatch_tokens
    s = make(6, 2, 3, 5, F32, F32, 4)
    moved, y, dx, dr, dw = all_passes(s)
    dy, dm = s["dy"].double(), s["drows"].double()
    loss = lambda x, r, w: float((combine_tokens(r, w, s["order"]).double() * dy).sum() +  # noqa: E731
                                 (dispatch_tokens(x, s["order"]).double() * dm).sum())
    base = loss(s["x"], s["rows"], s["w"])
    for name, grad in (("x", dx), ("rows", dr), ("w", dw)):
        for i in range(grad.numel()):
            t = {n: s[n].clone() for n in ("x", "rows", "w")}
            t[name].view(-1)[i] += 1.0
            assert abs(loss(t["x"], t["rows"], t["w"]) - base - grad.flatten()[i].item()) <= 1e-5


def test_second_derivatives_are_refused():
    from muon_sr_amd import combine_tokens, dispatch_tokens
    s = make(9, 2, 3, 16, F32, F32, 9)
    x, w = s["x"].requires_grad_(True), s["w"].requires_grad_(True)
    y = combine_tokens(dispatch_tokens(x, s["order"]), w, s["order"])
    (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


def test_only_what_is_wanted():
    """Frozen weights, or frozen rows."""
    from muon_sr_amd import combine_tokens
    s = make(50, 2, 4, 72, BF16, BF16, 5)
    full = all_passes(s)
    r, w = s["rows"].clone().requires_grad_(True), s["w"].clone()
    combine_tokens(r, w, s["order"]).backward(s["dy"])
    assert torch.equal(r.grad, full[3])
    r, w = s["rows"].clone(), s["w"].clone().requires_grad_(True)
    combine_tokens(r, w, s["order"]).backward(s["dy"])
    assert torch.equal(w.grad, full[4])


def test_rows_beyond_2_31_elements():
    """Byte and element offsets past 32 bits: 2^21 + 2 rows of 1026 elements."""
    from muon_sr_amd import combine_tokens, dispatch_tokens, order_tokens
    tokens, d = (1 << 20) + 1, 1026
    ids = torch.randint(0, 4, (tokens, 2), generator=gen(6), device=DEV)
    order = order_tokens(ids, 4)
    x = torch.randn((tokens, d), generator=gen(7), device=DEV, dtype=BF16)
    rows = dispatch_tokens(x, order)
    w = torch.tensor([0.25, 0.5], device=DEV).expand(tokens, 2)
    y = combine_tokens(rows, w, order)
    # 0.25 x + 0.5 x = 0.75 x, exact in fp32 before its one rounding
    assert torch.equal(y, (x.float() * 0.75).to(BF16))


def test_refusals():
    from muon_sr_amd import _lib, combine_tokens, dispatch_tokens, order_tokens
    s = make(8, 2, 4, 16, BF16, F32, 8)
    o = s["order"]
    ids = torch.zeros(8, 2, dtype=torch.int64, device=DEV)
    for call in (lambda: order_tokens(ids.float(), 4), lambda: order_tokens(ids.view(-1), 4), lambda: order_tokens(ids.cpu(), 4),
                 lambda: order_tokens(ids[:, :0], 4), lambda: dispatch_tokens(s["x"][:7], o),
                 lambda: dispatch_tokens(s["x"].half(), o), lambda: dispatch_tokens(s["x"].cpu(), o),
                 lambda: combine_tokens(s["rows"][:15], s["w"], o), lambda: combine_tokens(s["rows"], s["w"].half(), o),
                 lambda: combine_tokens(s["rows"], s["w"][:, :1], o),
                 lambda: dispatch_tokens(s["x"], (o.offsets.long(), o.position, o.source))):
        with pytest.raises(ValueError):
            call()
    for experts in (-1, 0, 1025):
        with pytest.raises(_lib.MuonSRLibraryError, match="experts|bad arguments"):
            order_tokens(ids, experts)
