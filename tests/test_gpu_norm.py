"""Layer norm and its gradients against 64-bit evaluations.

Bounds, with u = 2^-24, s the type's unit roundoff, and a sum of n fp32 terms off by at most n u sum|terms| (any order; the
kernel's has far fewer additions one after the other).  d elements to a row:
    mean    em = (d + 2) u mean|x|
    x - mean, and so the variance: relative (d + 8) u, and em^2; rstd r: relative er = (d + 8) u + em^2 / var' (var' = var + eps)
    h       eh = r (em + u |x - mean|) + |h| (er + 2 u)
    y       |w| eh + 2 u (|h w| + |b|) + s |y|
    q = dy w: u |q|;  mean(q): e1 = (d + 3) u mean|q|;  mean(q h): e2 = (d + 4) u mean|q h| + mean(|q| eh)
    dx      r (e1 + |h| e2 + eh (|mean(q h)| + e2) + 4 u (|q| + |mean q| + |h mean(q h)|)) + (er + 2 u) |dx| + s |dx|
    dw, db  (rows + 8) u sum|terms| + sum |dy| eh + s |value|"""
import pytest
import torch

from _gpu import DEV, need_gpu

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
UNIT = {BF16: 2.0 ** -8, F32: U}
EPS = 1e-5


@pytest.fixture(scope="module", autouse=True)
def L():
    return need_gpu()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make(rows, d, dtype, wdtype, seed, offset=0.5):
    g = gen(seed)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    x = (r(rows, d) * (torch.rand((rows, 1), generator=g, device=DEV) + 0.1) + offset * r(d)).to(dtype)
    return x, (1 + 0.1 * r(d)).to(wdtype), (0.1 * r(d)).to(wdtype), r(rows, d).to(dtype)


def exact(x, w, b, dy, eps=EPS):
    """(value, bound without the stored value's rounding) of y, dx, dw, db."""
    n, d = x.shape
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    mean = x.mean(1, keepdim=True)
    em = (d + 2) * U * x.abs().mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True) + eps
    r = var.rsqrt()
    er = (d + 8) * U + em ** 2 / var
    h = (x - mean) * r
    eh = r * (em + U * (x - mean).abs()) + h.abs() * (er + 2 * U)
    y = (h * w + b, w.abs() * eh + 2 * U * ((h * w).abs() + b.abs()))
    q = dy * w
    m1, m2 = q.mean(1, keepdim=True), (q * h).mean(1, keepdim=True)
    e1 = (d + 3) * U * q.abs().mean(1, keepdim=True)
    e2 = (d + 4) * U * (q * h).abs().mean(1, keepdim=True) + (q.abs() * eh).mean(1, keepdim=True)
    dx = r * (q - m1 - h * m2)
    ex = r * (e1 + h.abs() * e2 + eh * (m2.abs() + e2) + 4 * U * (q.abs() + m1.abs() + (h * m2).abs())) + (er + 2 * U) * dx.abs()
    dw = ((dy * h).sum(0), (n + 8) * U * (dy * h).abs().sum(0) + (dy.abs() * eh).sum(0))
    db = (dy.sum(0), (n + 8) * U * dy.abs().sum(0))
    return y, (dx, ex), dw, db


def run(x, w, b, dy, eps=EPS):
    from muon_sr_amd import layer_norm
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    return [y.detach(), *torch.autograd.grad(y, [t for t in leaves if t is not None], dy)]


def near(got, want):
    value, bound = want
    unit = UNIT[got.dtype]
    assert got.shape == value.shape
    assert ((got.double() - value).abs() <= bound + unit * (value.abs() + bound) + 1e-37).all()


@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)], ids=["bf16", "bf16-fp32", "fp32", "fp32-bf16"])
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 8), (5, 3), (7, 384), (33, 512), (300, 1000), (67, 1024), (2, 1025), (129, 2048), (17, 2049),
                                    (65, 4096), (3, 5001), (12, 8192), (4, 8193), (5, 16384), (3, 20000), (700, 17), (5000, 64), (3001, 1400), (33001, 384),
                                    (1001, 128), (515, 256), (300, 12000), (260, 16383), (70, 16385), (65541, 200)])
def test_against_64_bits(rows, d, dtype, wdtype):
    x, w, b, dy = make(rows, d, dtype, wdtype, rows + d)
    for got, want in zip(run(x, w, b, dy), exact(x, w, b, dy)):
        near(got, want)


def test_without_weight_or_bias():
    x, w, b, dy = make(90, 300, BF16, F32, 1)
    one, zero = torch.ones_like(w), torch.zeros_like(b)
    for ww, bb in ((None, None), (w, None), (None, b)):
        got = run(x, ww, bb, dy)
        want = exact(x, one if ww is None else w, zero if bb is None else b, dy)
        picked = [want[0], want[1]] + ([want[2]] if ww is not None else []) + ([want[3]] if bb is not None else [])
        assert len(got) == len(picked)
        for a, b_ in zip(got, picked):
            near(a, b_)


def test_a_mean_far_from_zero_and_equal_rows():
    """fp32 rows around 1000 with deviations of 1e-2: a variance from sums of squares would have no digit left.  x minus any fp32
    number near it is exact, so y is as near as that of rows around 0: within 768 * 8 u of its size, below 1e-3 for |h| < 8.  Rows of
    equal elements give y = b."""
    g = gen(2)
    x = 1000 + 1e-2 * torch.randn((40, 768), generator=g, device=DEV)
    x[7] = 3.0
    _, w, b, dy = make(40, 768, F32, F32, 3)
    for got, want in zip(run(x, w, b, dy, 1e-6), exact(x, w, b, dy, 1e-6)):
        near(got, want)
    y = exact(x, w, b, dy, 1e-6)[0][0]
    keep = torch.arange(40, device=DEV) != 7
    assert ((run(x, w, b, dy, 1e-6)[0].double() - y)[keep].abs() <= 1e-3).all()
    for d in (768, 2048, 20000):
        y = run(torch.full((3, d), 3.0, device=DEV), torch.ones(d, device=DEV), torch.full((d,), 0.25, device=DEV), torch.ones((3, d), device=DEV))[0]
        assert torch.equal(y, torch.full((3, d), 0.25, device=DEV))


def test_non_finite_rows_stay_alone():
    for d in (200, 4000, 20000):
        x, w, b, dy = make(30, d, BF16, F32, 4)
        clean = run(x, w, b, dy)
        x[3, 5], x[11, d - 1] = float("nan"), float("inf")
        got = run(x, w, b, dy)
        others = torch.ones(30, dtype=torch.bool, device=DEV)
        others[[3, 11]] = False
        for k in (0, 1):
            assert torch.equal(got[k][others], clean[k][others]) and got[k][3].isnan().all() and got[k][11].isnan().any()
        assert torch.equal(got[3], clean[3])       # the bias's gradient reads dy alone


def test_strides_and_shapes():
    from muon_sr_amd import layer_norm
    for dtype in (BF16, F32):
        x, w, b, dy = make(60, 136, dtype, F32, 5)
        want = run(x, w, b, dy)
        wide = torch.zeros((2, 60, 200), dtype=dtype, device=DEV)
        wide[0, :, 3:139], wide[1, :, 1:137] = x, dy
        for xx, yy in ((wide[0, :, 3:139], wide[1, :, 1:137]), (x.t().contiguous().t(), dy.t().contiguous().t()),
                       (x.view(5, 12, 136), dy.view(5, 12, 136))):
            for a, v in zip(run(xx, w, b, yy), want):
                assert torch.equal(a.reshape(v.shape), v)
        gaps = torch.stack([w, w], 1)[:, 0]
        for a, v in zip(run(x, gaps, b, dy), want):
            assert torch.equal(a, v)
        one = dy[:1].expand(60, 136)
        assert all(torch.equal(p, q) for p, q in zip(run(x, w, b, one), run(x, w, b, one.contiguous())))
        vector = run(x[4], w, b, dy[4])
        assert torch.equal(vector[0], want[0][4]) and vector[1].shape == (136,)
        assert layer_norm(x[:0], w, b).shape == (0, 136)
        leaf = w.clone().requires_grad_(True)
        assert not torch.autograd.grad(layer_norm(x[:0], leaf, b), leaf, dy[:0])[0].any()


def test_only_some_gradients_wanted():
    from muon_sr_amd import layer_norm
    x, w, b, dy = make(100, 640, BF16, BF16, 6)
    want = run(x, w, b, dy)[1:]
    for k in range(3):
        leaves = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(layer_norm(*leaves), leaves[k], dy)[0], want[k])


def test_module_takes_the_place_of_torchs():
    import muon_sr_amd as M
    ours, theirs = M.LayerNorm(384, device=DEV, dtype=BF16), torch.nn.LayerNorm(384, device=DEV, dtype=BF16)
    theirs.load_state_dict(ours.state_dict())
    x, _, _, dy = make(50, 384, BF16, BF16, 7)
    for got, want in ((ours(x), theirs(x.float().to(BF16))),):
        assert ((got.double() - want.double()).abs() <= 2 * 2.0 ** -7 * want.double().abs() + 1e-2).all()
    y = ours(x)
    y.backward(dy)
    assert ours.weight.grad.dtype == BF16 and ours.bias.grad.shape == (384,)
    assert M.LayerNorm(16, elementwise_affine=False, device=DEV)(x[:, :16]).shape == (50, 16)
    for bad in (lambda: M.LayerNorm((4, 8)), lambda: ours(x[:, :16]), lambda: M.layer_norm(x, ours.weight[:5]),
                lambda: M.layer_norm(x, ours.weight, ours.bias.float()), lambda: M.layer_norm(x.half()), lambda: M.layer_norm(x.cpu())):
        with pytest.raises(ValueError):
            bad()


def test_gradient_is_that_of_differences():
    """(f(x + t v) - f(x - t v)) / 2t of f = <y, dy> in the operator's own fp32, against <dx, v>.  Along v, f is smooth with a
    third derivative below 50 (rstd^3 |v|^3 |dy w|, rows of unit deviation, |v| = 1 to a row): t^2 / 6 of it, and the values' rounding,
    2 d u (|f| terms) / 2t."""
    x, w, b, dy = make(8, 96, F32, F32, 8, offset=0.0)
    x = (x - x.mean(1, keepdim=True)) / x.std(1, keepdim=True)
    from muon_sr_amd import layer_norm
    dx = run(x, w, b, dy)[1].double()
    t = 2.0 ** -6
    f = lambda v: (layer_norm(v, w, b).double() * dy.double()).sum(1)  # noqa: E731
    for k in range(5):
        v = torch.randn((8, 96), generator=gen(20 + k), device=DEV)
        v = v / v.norm(dim=1, keepdim=True)
        hi, lo = x + t * v, x - t * v
        diff = (f(hi) - f(lo)) / (2 * t)
        step = (hi.double() - lo.double()) / (2 * t)
        terms = (layer_norm(x, w, b).double() * dy.double()).abs().sum(1)
        scale = (dy.double() * w.double()).norm(dim=1)
        tol = t * t / 6 * 50 * scale + 2 * 96 * U * terms / t
        assert ((diff - (dx * step).sum(1)).abs() <= tol).all()


def test_same_call_same_bits():
    x, w, b, dy = make(3000, 1000, BF16, F32, 9)
    a = run(x, w, b, dy)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(a, run(x, w, b, dy)))


def exact_far(x, w, b, dy, eps, depth):
    """As `exact`, for rows whose mean is far from zero and held as two numbers, m and c.  A sum has at most `depth` additions one after the
    other (and a division), so m is off by em = depth u mean|x|.  z = x - m is exact (x and m are within a factor of 2 of one another) and at most
    Z = |x - mean| + em; c = mean(z) is off by ec = depth u mean Z, z - c by ec + u (Z + em + ec).  mean(z^2) - c^2 is off by
    (depth + 4) u mean Z^2 + 2 (em + ec) (ec + u em), the variance's relative error twice that of rstd, which adds 4 u."""
    n, d = x.shape
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    mean = x.mean(1, keepdim=True)
    assert (x.amax(1) < 2 * x.amin(1)).all()
    em = depth * U * x.abs().mean(1, keepdim=True)
    Z = (x - mean).abs() + em
    ec = depth * U * Z.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True) + eps
    r = var.rsqrt()
    er = ((depth + 4) * U * Z.square().mean(1, keepdim=True) + 2 * (em + ec) * (ec + U * em)) / var + 4 * U
    h = (x - mean) * r
    eh = r * (ec + U * (Z + em + ec)) + h.abs() * (er + 2 * U)
    y = (h * w + b, w.abs() * eh + 2 * U * ((h * w).abs() + b.abs()))
    q = dy * w
    m1, m2 = q.mean(1, keepdim=True), (q * h).mean(1, keepdim=True)
    e1 = (depth + 1) * U * q.abs().mean(1, keepdim=True)
    e2 = (depth + 2) * U * (q * h).abs().mean(1, keepdim=True) + (q.abs() * eh).mean(1, keepdim=True)
    dx = r * (q - m1 - h * m2)
    ex = r * (e1 + h.abs() * e2 + eh * (m2.abs() + e2) + 4 * U * (q.abs() + m1.abs() + (h * m2).abs())) + (er + 2 * U) * dx.abs()
    dw = ((dy * h).sum(0), (n + 8) * U * (dy * h).abs().sum(0) + (dy.abs() * eh).sum(0))
    db = (dy.sum(0), (n + 8) * U * dy.abs().sum(0))
    return y, (dx, ex), dw, db


@pytest.mark.parametrize("d", [40, 200, 768, 4096, 8000, 20000])
def test_gradients_of_rows_far_from_zero(d):
    """fp32 rows around 1000 with deviations of 1e-2, in every way that a row is held: their h, and with it the gradients, keep the digits that
    y keeps.  A mean rounded to one number would be off by 2^-15, and h by 3e-3 with it.  One lane adds up at most 32 elements (of a long row d / 256,
    4 at a time), a wave 6 times two, and 16 waves their sums; the bounds are below 3e-4 of the values' size, so such a mean does not pass."""
    g = gen(30 + d)
    x = 1000 + 1e-2 * torch.randn((40, d), generator=g, device=DEV)
    _, w, b, dy = make(40, d, F32, F32, 31)
    depth = (32 if d <= 16384 else d // 256 + 4) + 6 + 16
    for got, want in zip(run(x, w, b, dy, 1e-6), exact_far(x, w, b, dy, 1e-6, depth)):
        near(got, want)
        assert torch.linalg.norm(want[1]) <= 3e-4 * torch.linalg.norm(want[0])


@pytest.mark.parametrize("rows,d", [(600000, 4096), (120000, 20000)])
def test_more_than_2_31_elements(rows, d):
    """The last rows of y and dx are those of a call of them alone, bit for bit; dw and db are the sums over all rows."""
    g = gen(50)
    x, dy = (torch.randn((rows, d), generator=g, device=DEV, dtype=BF16) for _ in range(2))
    _, w, b, _ = make(1, d, BF16, F32, 51)
    y, dx, dw, db = run(x, w, b, dy)
    last = slice(rows - 700, rows)
    alone = run(x[last], w, b, dy[last])
    assert torch.equal(y[last], alone[0]) and torch.equal(dx[last], alone[1])
    del y, dx
    sums = [torch.zeros(d, dtype=torch.float64, device=DEV) for _ in range(4)]
    for i in range(0, rows, 10000):
        _, _, (v, e), (u, f) = exact(x[i:i + 10000], w, b, dy[i:i + 10000])
        for s, t in zip(sums, (v, e, u, f)):
            s += t
    near(dw, (sums[0], sums[1] * rows / 10000))      # (the bound of the sums is rows u times the terms')
    near(db, (sums[2], sums[3] * rows / 10000))
