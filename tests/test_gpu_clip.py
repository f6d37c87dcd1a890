"""The global gradient norm and clipping against 64-bit evaluations.

The norm's sums are in 64 bits (relative error n 2^-53), so the fp32 result is within one
rounding, 2^-24, of the exact norm; 2^-23 is asserted.  Given the norm, every clipped
element is defined exactly: round(f32(g) * c) with c = max_norm / (norm + 1e-6) in fp32, which
torch on the CPU evaluates with the same IEEE operations: those are compared bit for bit."""
import math

import pytest
import torch

from _gpu import DEV, need_gpu

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
TILE = 8192


@pytest.fixture(scope="module", autouse=True)
def L():
    return need_gpu()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(n, dtype, seed, std=1e-2):
    return (torch.randn(n, generator=gen(seed), device=DEV, dtype=F32) * std).to(dtype)


def norm64(grads, p):
    v = [g.detach().cpu().double().abs().flatten() for g in grads if g.numel()]
    if not v:
        return 0.0
    if p == math.inf:
        return max(x.max().item() for x in v)
    return sum((x ** p).sum().item() for x in v) ** (1.0 / p)


def coefficient(norm, max_norm):
    """c as the kernel forms it, from the norm it returned."""
    one = torch.tensor(max_norm, dtype=F32) / (norm.cpu() + torch.tensor(1e-6, dtype=F32))
    return torch.where(one >= 1.0, torch.tensor(1.0), one)


def expect(g, norm, max_norm, dtype):
    return (g.cpu().float() * coefficient(norm, max_norm)).to(dtype)


def same(a, b):
    a, b = a.detach().cpu().flatten(), b.detach().cpu().flatten()
    assert a.dtype == b.dtype and a.shape == b.shape
    it = torch.int16 if a.dtype == BF16 else torch.int32
    nan = torch.isnan(a.float()) & torch.isnan(b.float())
    assert bool(((a.view(it) == b.view(it)) | nan).all())


SIZES = {
    "one": [1],
    "empties": [0, 3, 0, 0, 8, 0],
    "around_a_tile": [TILE - 1, TILE, TILE + 1, 2 * TILE + 7, 8, 9],
    "many_tensors": [17 * i % 1031 for i in range(300)],
    "beyond_the_grid": [2049 * TILE + 3, 5],
}


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("sizes", list(SIZES))
def test_norm_and_clip(sizes, dtype, p):
    from muon_sr_amd import clip_grads, grad_norm
    grads = [randn(n, dtype, 10 + i, 1e-2 * (1 + i % 3)) for i, n in enumerate(SIZES[sizes])]
    ref = norm64(grads, p)
    got = grad_norm(grads, p)
    assert got.dtype == F32 and got.shape == ()
    assert abs(got.item() - ref) <= 2.0 ** -23 * ref
    before = [g.clone() for g in grads]
    norm = clip_grads(grads, 0.37 * ref, p)
    assert norm.item() == got.item()
    for g, b in zip(grads, before):
        same(g, expect(b, norm, 0.37 * ref, dtype))
    # out of place, into bf16; the gradients stay
    outs = [torch.full_like(b, 7.0, dtype=BF16) for b in before]
    kept = [b.clone() for b in before]
    norm = clip_grads(before, 0.37 * ref, p, out=outs)
    for b, k, o in zip(before, kept, outs):
        same(b, k)
        same(o, expect(k, norm, 0.37 * ref, BF16))


def test_norm_is_the_same_bits_every_time():
    from muon_sr_amd import grad_norm
    grads = [randn(100003 + i, BF16, i) for i in range(40)]
    first = grad_norm(grads).item()
    assert all(grad_norm(grads).item() == first for _ in range(5))


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_nothing_to_cut(p):
    """A norm below the bound: c = 1, and out of place is a copy."""
    from muon_sr_amd import clip_grads
    grads = [randn(1003, BF16, 1), torch.zeros(12, dtype=BF16, device=DEV)]
    kept = [g.clone() for g in grads]
    clip_grads(grads, 1e6, p)
    for g, k in zip(grads, kept):
        same(g, k)
    outs = [torch.empty_like(g) for g in grads]
    clip_grads(grads, 1e6, p, out=outs)
    for o, k in zip(outs, kept):
        same(o, k)


def test_zero_gradients_and_zero_bound():
    from muon_sr_amd import clip_grads
    z = torch.zeros(100, dtype=BF16, device=DEV)
    assert clip_grads([z], 1.0).item() == 0.0
    assert not z.any()
    g = randn(100, BF16, 1)
    assert clip_grads([g], 0.0).item() > 0.0
    assert not g.any()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("scale", [1e30, 1e-30])
def test_squares_out_of_fp32_range(scale, dtype):
    from muon_sr_amd import clip_grads
    g = (torch.randn(5000, generator=gen(3), device=DEV) * scale).to(dtype)
    ref, kept = norm64([g], 2.0), g.clone()
    norm = clip_grads([g], 0.5 * ref)
    assert abs(norm.item() - ref) <= 2.0 ** -23 * ref
    same(g, expect(kept, norm, 0.5 * ref, dtype))


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_non_finite(bad, p):
    """As torch: a NaN norm makes everything NaN; an infinite one makes finite elements 0 and infinite ones NaN."""
    from muon_sr_amd import clip_grad_norm_, clip_grads
    g, h = randn(9001, BF16, 4), randn(33, BF16, 5)
    g[8999] = bad
    p_ = torch.nn.Parameter(torch.zeros_like(g))
    p_.grad = g.clone()
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grad_norm_([p_], 1.0, p, error_if_nonfinite=True)
    same(p_.grad, g)
    kept = [g.clone(), h.clone()]
    norm = clip_grads([g, h], 1.0, p)
    assert math.isnan(norm.item()) if math.isnan(bad) else norm.item() == math.inf
    for x, k in zip((g, h), kept):
        same(x, expect(k, norm, 1.0, BF16))
    assert bool(torch.isnan(h).all()) if math.isnan(bad) else not h.any()


def test_views_and_orders():
    """Unaligned, transposed (dense) and gapped gradients; outs of another order."""
    from muon_sr_amd import clip_grads, grad_norm
    base = randn(70001, BF16, 6)
    grads = [base[1:20002], base[20003:40003].view(200, 100).t(), randn(64 * 90, BF16, 7).view(64, 90)[:, 5:77],
             randn(24 * 35, BF16, 8).view(2, 12, 35).permute(2, 0, 1)]
    kept = [g.clone() for g in grads]
    ref = norm64(grads, 2.0)
    assert abs(grad_norm(grads).item() - ref) <= 2.0 ** -23 * ref
    outs = [torch.zeros(20001, dtype=BF16, device=DEV), torch.zeros(100, 200, dtype=BF16, device=DEV),
            torch.zeros(90, 64, dtype=BF16, device=DEV).t()[:, 5:77], torch.zeros(35, 2, 12, dtype=BF16, device=DEV)]
    norm = clip_grads(grads, 0.5 * ref, out=outs)
    for o, k in zip(outs, kept):
        same(o.contiguous(), expect(k, norm, 0.5 * ref, BF16))
    guard = (base[:1].clone(), base[20002:20003].clone(), base[40003:].clone())
    norm = clip_grads(grads, 0.5 * ref)
    for g, k in zip(grads, kept):
        same(g.contiguous(), expect(k, norm, 0.5 * ref, BF16))
    for a, b in zip(guard, (base[:1], base[20002:20003], base[40003:])):
        same(a, b)


def test_parameters_with_and_without_gradients():
    from muon_sr_amd import clip_grad_norm_
    ps = [torch.nn.Parameter(torch.zeros(100, 7, dtype=BF16, device=DEV)) for _ in range(3)]
    assert clip_grad_norm_(ps, 1.0).item() == 0.0
    ps[0].grad, ps[2].grad = randn(700, BF16, 1).view(100, 7), randn(700, BF16, 2).view(100, 7)
    kept = [ps[0].grad.clone(), ps[2].grad.clone()]
    # torch's own clipping in fp32 has the same norm to fp32 accuracy (700 * 2 terms: 2^-13 is far above their error)
    fp32 = [torch.nn.Parameter(torch.zeros(100, 7, device=DEV)) for _ in kept]
    for q, k in zip(fp32, kept):
        q.grad = k.float()
    want = torch.nn.utils.clip_grad_norm_(fp32, 0.1)
    norm = clip_grad_norm_(iter(ps), 0.1)
    assert abs(norm.item() - want.item()) <= 2.0 ** -13 * want.item()
    assert ps[1].grad is None
    for p, k in zip((ps[0], ps[2]), kept):
        same(p.grad, expect(k, norm, 0.1, BF16))


def test_more_than_2_31_elements():
    from muon_sr_amd import clip_grads
    n = (1 << 31) + 77
    g = torch.full((n,), 0.5, dtype=BF16, device=DEV)
    g[-1] = 3.0
    norm = clip_grads([g], 0.25 * math.sqrt(n) * 0.5)
    ref = math.sqrt(0.25 * (n - 1) + 9.0)
    assert abs(norm.item() - ref) <= 2.0 ** -23 * ref
    ends = torch.cat([g[:3], g[(1 << 31) - 2:(1 << 31) + 2], g[-2:]])
    kept = torch.full((9,), 0.5, dtype=BF16)
    kept[-1] = 3.0
    same(ends, expect(kept, norm, 0.25 * math.sqrt(n) * 0.5, BF16))
    assert g.min().item() == g.flatten()[0].item()


def test_refusals():
    from muon_sr_amd import _lib, clip_grads, grad_norm
    g, f = randn(64, BF16, 1), randn(64, F32, 1)
    for call in (lambda: grad_norm([g], 3.0), lambda: grad_norm([g.half()]), lambda: grad_norm([g.cpu()]),
                 lambda: clip_grads([g], 1.0, out=[f]), lambda: clip_grads([g], 1.0, out=[]),
                 lambda: clip_grads([g], 1.0, out=[g[:5]]), lambda: clip_grads([g, g.cpu()], 1.0)):
        with pytest.raises(ValueError):
            call()
    kept = g.clone()
    for grads, out in (([g, g], None), ([g[:40], g[8:]], None), ([g[:32]], [g[16:48]])):
        with pytest.raises(_lib.MuonSRLibraryError, match="overlap"):
            clip_grads(grads, 1e-3, out=out)
    same(g, kept)
    sparse = torch.sparse_coo_tensor([[0, 2]], torch.ones(2, device=DEV, dtype=BF16), (4,))
    for call in (lambda: grad_norm([sparse]), lambda: clip_grads([g, sparse], 1.0)):
        with pytest.raises(RuntimeError):
            call()
    same(g, kept)
    # gradients that require gradients themselves (a graph of the backward pass was made)
    h = g.clone().requires_grad_(True)
    assert clip_grads([h], 1e-3).item() == grad_norm([kept]).item() and not torch.equal(h, kept)
    # reading the same memory twice is no conflict
    assert abs(grad_norm([g, g]).item() - math.sqrt(2) * norm64([g], 2.0)) <= 2.0 ** -22 * norm64([g], 2.0)


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("where", [None, 3, 150, 400])
def test_lists_of_several_launches(where, p):
    """Launches of few, many, and few work-groups again, whose partial sums join; a NaN in any of them reaches the norm."""
    from muon_sr_amd import clip_grads, grad_norm
    grads = [randn(n, BF16, 20 + i, 1e-2 * (1 + i % 5)) for i, n in enumerate([5] * 112 + [90001] * 112 + [9, 3000] * 100)]
    ref = norm64(grads, p)
    if where is not None:
        grads[where][-1] = math.nan
    got, kept = grad_norm(grads, p), [g.clone() for g in grads]
    assert math.isnan(got.item()) if where is not None else abs(got.item() - ref) <= 2.0 ** -23 * ref
    norm = clip_grads(grads, 0.37 * ref, p)
    same(norm.view(1), got.view(1))
    for g, k in zip(grads, kept):
        same(g, expect(k, norm, 0.37 * ref, BF16))
