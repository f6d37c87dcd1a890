"""The experts' products against plain 64-bit evaluations.

Bound.  bf16 products are exact in fp32; a sum of K of them in fp32, in any order, is within
K 2^-24 sum|terms| of the exact one (first order), and storing as bf16 (8 significant bits) adds 2^-8 of the value:
|got - exact| <= 2^-8 |exact| + 2 K 2^-24 sum|terms|.  The accumulation is compared bit for bit with
the stored product followed by msr_sr_accum."""
import ctypes
import random

import pytest
import torch

from _gpu import DEV, check, need_gpu, stream

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def L():
    return need_gpu()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def offsets_of(counts):
    off = torch.zeros(len(counts) + 1, dtype=torch.int32)
    off[1:] = torch.tensor(counts).cumsum(0)
    return off.to(DEV)


def make(counts, spare, fout, fin, seed):
    g = gen(seed)
    rows = sum(counts) + spare
    r = lambda *s: torch.randn(s, generator=g, device=DEV, dtype=BF16)  # noqa: E731
    return dict(off=offsets_of(counts), x=r(rows, fin), w=r(len(counts), fout, fin) * 0.05, dy=r(rows, fout))


def plain(s, what, absolute=False):
    """The operator in 64 bits, or (absolute) the sums of the terms' magnitudes."""
    f = (lambda t: t.double().abs()) if absolute else (lambda t: t.double())
    x, w, dy, off = f(s["x"]), f(s["w"]), f(s["dy"]), s["off"].tolist()
    out = torch.zeros({"y": dy.shape, "dx": x.shape, "dw": w.shape}[what], dtype=torch.float64, device=DEV)
    for e in range(len(off) - 1):
        lo, hi = off[e], off[e + 1]
        if what == "y":
            out[lo:hi] = x[lo:hi] @ w[e].t().contiguous()
        elif what == "dx":
            out[lo:hi] = dy[lo:hi] @ w[e]
        else:
            out[e] = dy[lo:hi].t().contiguous() @ x[lo:hi]
    return out


def near(got, s, what, K):
    exact, terms = plain(s, what), plain(s, what, True)
    bound = 2.0 ** -8 * exact.abs() + 2 * K * 2.0 ** -24 * terms
    assert got.dtype == BF16 and bool(((got.double() - exact).abs() <= bound).all())


def passes(s, x=None, dy=None):
    from muon_sr_amd import expert_linear
    x = (s["x"] if x is None else x).detach().requires_grad_(True)
    w = s["w"].detach().requires_grad_(True)
    y = expert_linear(x, w, s["off"])
    return (y, *torch.autograd.grad(y, (x, w), s["dy"] if dy is None else dy))


COUNTS = {
    "one_row": [1],
    "none": [0, 0, 0],
    "empty_between": [0, 5, 0, 0, 130, 1, 0],
    "around_tiles": [63, 64, 65, 127, 128, 129, 255, 256, 257],
    "one_has_all": [0] * 20 + [900] + [0] * 10,
    "many_small": [i * 7 % 23 for i in range(200)],
    "uneven": [700, 3, 0, 41, 1200, 17],
    "most_experts": [i * 5 % 7 for i in range(1024)],
}


@pytest.mark.parametrize("spare", [0, 37])
@pytest.mark.parametrize("fout,fin", [(8, 8), (24, 16), (136, 264), (256, 128), (520, 72)])
@pytest.mark.parametrize("counts", list(COUNTS))
def test_products(L, counts, fout, fin, spare):
    c = COUNTS[counts]
    s = make(c, spare, fout, fin, fout + fin + spare)
    y, dx, dw = passes(s)
    near(y, s, "y", fin)
    near(dx, s, "dx", fout)
    near(dw, s, "dw", max(c))
    n = sum(c)
    assert not y[n:].any() and not dx[n:].any()
    assert all(torch.equal(a, b) for a, b in zip((y, dx, dw), passes(s)))


@pytest.mark.parametrize("counts,fout,fin", [([512, 1024, 300, 212], 768, 1024), ([3000, 100, 1003], 1024, 2048),
                                             ([256] * 16, 512, 384), ([20] * 64, 1536, 384)])
def test_products_of_ordinary_layers(L, counts, fout, fin):
    s = make(counts, 5, fout, fin, 3)
    y, dx, dw = passes(s)
    near(y, s, "y", fin)
    near(dx, s, "dx", fout)
    near(dw, s, "dw", max(counts))


@pytest.mark.parametrize("counts,fout,fin,tiles", [([41, 0, 130, 29, 0, 99, 1], 264, 136, [64, 64, 64, 64]),
                                                   ([1201, 0, 900, 7, 893], 1544, 2056, [128, 128, 128, 128]),
                                                   ([1013, 987], 4096, 4096, [256, 256, 256, 256]),
                                                   ([1500, 1, 1499], 2056, 4104, [128, 256, 256, 128]),
                                                   ([70, 0, 133], 136, 4104, [63, 64, 64, 64]),
                                                   ([70, 0, 133], 4168, 136, [64, 63, 64, 64]),
                                                   ([1], 4168, 8200, [63, 63, 128, 128])])
def test_every_tile(L, counts, fout, fin, tiles):
    """Each product in each of its tiles (63: 64 with K split; features and groups that end inside them), the
    accumulation against
    the stored product whatever its tile: the same products in the same order."""
    from muon_sr_amd import _lib, experts_wgrad_sr_accum
    s = make(counts, 9, fout, fin, 4)
    rows, E, t, split = s["x"].shape[0], len(counts), ctypes.c_int32(), ctypes.c_int32()
    for product, tile in enumerate(tiles):
        check(L, L.msr_experts_tile(product, rows, E, fin, fout, ctypes.byref(t), ctypes.byref(split)))
        assert t.value - split.value == tile
    y, dx, dw = passes(s)
    near(y, s, "y", fin)
    near(dx, s, "dx", fout)
    near(dw, s, "dw", max(counts))
    assert not y[rows - 9:].any() and not dx[rows - 9:].any()
    w, want = torch.nn.Parameter(s["w"].clone()), torch.zeros_like(dw)
    for micro in range(2):
        experts_wgrad_sr_accum(w, s["x"], s["dy"], s["off"], seed=99 + micro)
        check(L, L.msr_sr_accum(want.data_ptr(), dw.data_ptr(), 0, dw.numel(), 99 + micro, int(micro == 0), _lib.noise_mode(),
                                None, stream()))
        assert torch.equal(w.acc_grad, want)


def test_no_rows(L):
    s = make([0, 0], 0, 16, 24, 1)
    y, dx, dw = passes(s)
    assert y.shape == (0, 16) and dx.shape == (0, 24) and dw.shape == (2, 16, 24) and not dw.any()


@pytest.mark.parametrize("mode", ["philox8", "triton"])
@pytest.mark.parametrize("counts,fout,fin", [([0, 5, 130, 1], 24, 16), ([300, 17, 700], 264, 136), ([64, 64], 256, 256),
                                             ([2000, 0, 513], 512, 640)])
def test_accumulation_is_the_stored_product_accumulated(L, counts, fout, fin, mode):
    from muon_sr_amd import _lib, experts_wgrad_sr_accum, get_sr_noise, set_sr_noise
    s = make(counts, 3, fout, fin, 9)
    dw = passes(s)[2]
    before = get_sr_noise()
    set_sr_noise(mode)
    try:
        for seed in (12345, 0x9ABCDEF0):
            w = torch.nn.Parameter(s["w"].clone())
            want = torch.zeros_like(dw)
            for micro in range(3):       # the first one creates the buffer
                experts_wgrad_sr_accum(w, s["x"], s["dy"], s["off"], seed=seed + micro)
                check(L, L.msr_sr_accum(want.data_ptr(), dw.data_ptr(), 0, dw.numel(), seed + micro, int(micro == 0),
                                        _lib.noise_mode(), None, stream()))
                assert torch.equal(w.acc_grad, want)
    finally:
        set_sr_noise(before)


def test_accumulation_with_injected_noise(L):
    s = make([40, 0, 100], 0, 64, 72, 10)
    dw, acc = passes(s)[2], torch.randn(3, 64, 72, generator=gen(1), device=DEV, dtype=BF16)
    want = acc.clone()
    noise = torch.randint(0, 65536, (acc.numel(),), generator=gen(2), device=DEV).to(torch.uint16)
    check(L, L.msr_experts_wgrad_sr_accum(acc.data_ptr(), s["x"].data_ptr(), 72, s["dy"].data_ptr(), 64, s["off"].data_ptr(),
                                          140, 3, 72, 64, 0, 0, 2, noise.data_ptr(), stream()))
    check(L, L.msr_sr_accum(want.data_ptr(), dw.data_ptr(), 0, dw.numel(), 0, 0, 2, noise.data_ptr(), stream()))
    assert torch.equal(acc, want)


def test_module_accumulates_as_the_hook_does(L):
    """SRExperts with the accumulator's hooks gives the acc_grad that expert_linear and the hook give with
    the same random state, over micro-batches; reassign_grad_buffer hands it to the optimizer."""
    from muon_sr_amd import SRExperts, TritonSRAccumulator, expert_linear
    s = make([100, 0, 60, 29], 2, 48, 64, 11)
    layer, plain_ = SRExperts(4, 64, 48, device=DEV), torch.nn.Module()
    plain_.weight = torch.nn.Parameter(layer.weight.detach().clone())
    TritonSRAccumulator.assign_hooks(layer)
    TritonSRAccumulator.assign_hooks(plain_)
    for run in (lambda x: layer(x, s["off"]), lambda x: expert_linear(x, plain_.weight, s["off"])):
        random.seed(5)
        for _ in range(3):
            run(s["x"].clone().requires_grad_(True)).backward(s["dy"])
    assert layer.weight.grad is None and plain_.weight.grad is None
    assert torch.equal(layer.weight.acc_grad, plain_.weight.acc_grad)
    TritonSRAccumulator.reassign_grad_buffer(layer)
    assert layer.weight.grad.shape == (4, 48, 64) and not hasattr(layer.weight, "acc_grad")


def test_rows_outside_the_groups_reach_nothing(L):
    """NaN and infinity in spare rows, and in one expert's rows, stay there."""
    s = make([70, 33, 0, 90], 40, 64, 96, 12)
    y, dx, dw = passes(s)
    s["x"][193:] = float("nan")
    s["dy"][193:] = float("inf")
    assert all(torch.equal(a, b) for a, b in zip((y, dx, dw), passes(s)))
    s["x"][80] = float("nan")            # expert 1
    s["dy"][80] = float("inf")
    y2, dx2, dw2 = passes(s)
    keep = torch.arange(233, device=DEV) != 80
    assert torch.equal(y2[keep], y[keep]) and torch.equal(dx2[keep], dx[keep])
    for e in (0, 2, 3):
        assert torch.equal(dw2[e], dw[e])
    assert not torch.isfinite(y2[80]).any() and not torch.isfinite(dw2[1]).any()
    # an expert's weights do not meet another's rows
    s = make([70, 33, 0, 90], 40, 64, 96, 12)
    s["w"][2] = float("nan")
    y3, dx3, _ = passes(s)
    assert torch.equal(y3, y) and torch.equal(dx3, dx)


def test_strides_and_alignment(L):
    s = make([50, 3, 77], 6, 40, 56, 13)
    want = passes(s)
    wide = torch.full((136, 160), float("nan"), dtype=BF16, device=DEV)
    for first in (0, 8, 3):
        x, dy = wide[:, first:first + 56], wide.clone()[:, 80 + first:120 + first]
        x.copy_(s["x"])
        dy.copy_(s["dy"])
        assert all(torch.equal(a, b) for a, b in zip(want, passes(s, x, dy)))
        wide.fill_(float("nan"))
    assert all(torch.equal(a, b) for a, b in zip(want, passes(s, s["x"].t().contiguous().t(), s["dy"].t().contiguous().t())))


def test_offsets_are_clamped_to_the_rows(L):
    s = make([50, 30], 0, 16, 24, 14)
    want = passes(s)
    s["off"][2] = 1000
    assert all(torch.equal(a, b) for a, b in zip(want, passes(s)))


def test_offsets_that_do_not_ascend_stay_inside(L):
    """Not a valid order: the results mean nothing, but every row and weight that is read or written is the call's."""
    s = make([50, 30, 20], 0, 72, 136, 18)
    for bad in ([0, 90, 10, 100], [0, -5, 1000, 60], [7, 100, 0, 100], [0, 100, 100, -3]):
        s["off"] = torch.tensor(bad, dtype=torch.int32, device=DEV)
        y, dx, dw = passes(s)
        assert y.shape == (100, 72) and dx.shape == (100, 136) and dw.shape == (3, 72, 136)
    torch.cuda.synchronize()


def test_gradients_against_differences(L):
    """The products are linear in each operand, so differences at unit steps on small whole numbers (exact in
    bf16 and fp32) are the gradients, exactly."""
    from muon_sr_amd import expert_linear
    s = make([3, 0, 4], 1, 8, 8, 15)
    for n in ("x", "w", "dy"):
        s[n] = torch.randint(-3, 4, s[n].shape, generator=gen(16), device=DEV).to(BF16)
    y, dx, dw = passes(s)
    loss = lambda x, w: float((expert_linear(x, w, s["off"]).double() * s["dy"].double()).sum())  # noqa: E731
    base = loss(s["x"], s["w"])
    for name, grad in (("x", dx), ("w", dw)):
        for i in range(0, grad.numel(), 5):
            t = {n: s[n].clone() for n in ("x", "w")}
            t[name].view(-1)[i] += 1.0
            assert loss(t["x"], t["w"]) - base == grad.flatten()[i].item()


def test_weights_beyond_2_31_elements(L):
    """Experts whose weights start past 2^31 elements, and their accumulation's noise offsets."""
    from muon_sr_amd import _lib, experts_wgrad_sr_accum
    E, o, i = 9, 16384, 16384
    x = torch.randn((20, i), generator=gen(1), device=DEV, dtype=BF16)
    dy = torch.randn((20, o), generator=gen(2), device=DEV, dtype=BF16)
    off = offsets_of([0] * 8 + [20])
    w = torch.nn.Parameter(torch.zeros((E, o, i), dtype=BF16, device=DEV))
    with torch.no_grad():
        w[8].copy_(torch.randn((o, i), generator=gen(3), device=DEV, dtype=BF16) * 0.05)
    s = dict(off=offsets_of([20]), x=x, w=w.detach()[8:], dy=dy)
    from muon_sr_amd import expert_linear
    xg = x.clone().requires_grad_(True)
    y = expert_linear(xg, w, off)
    (dx,) = torch.autograd.grad(y, xg, dy)
    near(y, s, "y", i)
    near(dx, s, "dx", o)
    experts_wgrad_sr_accum(w, x, dy, off, seed=7)
    assert not w.acc_grad[:8].any()
    alone = torch.nn.Parameter(s["w"].clone())
    dw = passes(dict(s, w=alone.detach()))[2]
    want = torch.zeros_like(w.acc_grad)
    want[8] = dw[0]
    full = torch.zeros_like(want)
    check(L, L.msr_sr_accum(full.data_ptr(), want.data_ptr(), 0, full.numel(), 7, 1, _lib.noise_mode(), None, stream()))
    assert torch.equal(w.acc_grad, full)


def test_refusals(L):
    from muon_sr_amd import _lib, expert_linear, experts_wgrad_sr_accum
    s = make([4, 4], 0, 16, 24, 17)
    x, w, off, dy = s["x"], s["w"], s["off"], s["dy"]
    for call in (lambda: expert_linear(x.float(), w, off), lambda: expert_linear(x, w.float(), off),
                 lambda: expert_linear(x, w, off.long()), lambda: expert_linear(x, w, off[:-1]),
                 lambda: expert_linear(x[:, :16], w, off), lambda: expert_linear(x, w[:, :, :23], off),
                 lambda: expert_linear(x, w[0], off), lambda: expert_linear(x.cpu(), w, off),
                 lambda: expert_linear(x[:, :20].contiguous(), w[:, :, :20].contiguous(), off),
                 lambda: expert_linear(x, w.transpose(1, 2), off), lambda: experts_wgrad_sr_accum(w, x, dy[:7], off)):
        with pytest.raises(ValueError):
            call()
    rc = L.msr_experts_forward(x.data_ptr(), 24, w.data_ptr(), x.data_ptr(), off.data_ptr(), 8, 2, 24, 16, stream())
    assert rc == 1005 and b"overlap" in L.msr_last_error()
    assert L.msr_experts_dgrad(dy.data_ptr() + 2, 16, w.data_ptr(), x.data_ptr(), off.data_ptr(), 8, 2, 24, 16, stream()) == 1002
    assert _lib.lib().msr_experts_wgrad(w.data_ptr(), x.data_ptr(), 23, dy.data_ptr(), 16, off.data_ptr(), 8, 2, 24, 16,
                                        stream()) == 1001


def test_accumulators_of_another_kind_are_refused(L):
    """A buffer of another type, order or size is refused and stays as it was."""
    from muon_sr_amd import experts_wgrad_sr_accum
    s = make([4, 4], 0, 16, 24, 18)
    w = torch.nn.Parameter(s["w"])
    for buffer in (torch.zeros(2, 16, 24, device=DEV), torch.zeros(2, 24, 16, dtype=BF16, device=DEV).transpose(1, 2),
                   torch.zeros(2, 16, 16, dtype=BF16, device=DEV), torch.zeros(2, 16, 24, dtype=BF16)):
        w.acc_grad = buffer
        with pytest.raises(ValueError, match="acc_grad"):
            experts_wgrad_sr_accum(w, s["x"], s["dy"], s["off"])
        assert w.acc_grad is buffer and not buffer.any()


def test_a_refused_first_accumulation_leaves_no_buffer(L):
    from muon_sr_amd import experts_wgrad_sr_accum
    s = make([4, 4], 0, 16, 24, 19)
    w, fresh = torch.nn.Parameter(s["w"]), torch.nn.Parameter(s["w"].clone())
    with pytest.raises(ctypes.ArgumentError):
        experts_wgrad_sr_accum(w, s["x"], s["dy"], s["off"], seed="7")
    assert not hasattr(w, "acc_grad")
    for weight in (w, fresh):
        experts_wgrad_sr_accum(weight, s["x"], s["dy"], s["off"], seed=7)
    assert torch.equal(w.acc_grad, fresh.acc_grad)


def guarded(rows, cols, ld, fill, seed=None):
    """A [rows, cols] view of row stride ld, 64 elements into a buffer of `fill` that is longer by 4096; random
    values with a seed."""
    buffer = torch.full((rows * ld + 64 + 4096,), fill, dtype=BF16, device=DEV)
    view = buffer[64:64 + rows * ld].view(rows, ld)[:, :cols]
    if seed is not None:
        view.copy_(torch.randn((rows, cols), generator=gen(seed), device=DEV))
    return buffer, view


@pytest.mark.parametrize("pad", [0, 24])
@pytest.mark.parametrize("E,rows,fout,fin", [(3, 100, 72, 136), (63, 700, 72, 136), (64, 700, 72, 136), (65, 700, 136, 264),
                                             (1024, 2000, 24, 40), (1000, 300, 8, 8), (65, 9000, 520, 776), (5, 6000, 1544, 2056),
                                             (2, 3, 136, 4104), (2, 3, 4104, 136), (5, 9000, 2056, 3080)])
def test_no_offsets_reach_outside_the_operands(L, E, rows, fout, fin, pad):
    """Offsets that ascend and offsets that do not: with NaN around the inputs every output is finite, and what
    lies around the outputs is as it was."""
    g = torch.Generator().manual_seed(E + rows)
    _, x = guarded(rows, fin, fin + pad, float("nan"), 1)
    _, dy = guarded(rows, fout, fout + pad, float("nan"), 2)
    _, w = guarded(E * fout, fin, fin, float("nan"), 3)
    ascending = torch.randint(0, rows + 1, (E + 1,), generator=g).sort().values
    ascending[0] = 0
    for offsets in (ascending, ascending.flip(0), torch.randint(-50, rows + 50, (E + 1,), generator=g),
                    torch.where(torch.arange(E + 1) % 2 == 0, 0, rows), torch.full((E + 1,), -(1 << 31)),
                    torch.where(torch.arange(E + 1) % 2 == 0, -(1 << 31), (1 << 31) - 1)):
        off = offsets.to(torch.int32).to(DEV)
        outs = [guarded(n, c, c, 7.0) for n, c in ((rows, fout), (rows, fin), (E * fout, fin), (E * fout, fin))]
        y, dx, dw, acc = (v.data_ptr() for _, v in outs)
        op = (x.data_ptr(), fin + pad, dy.data_ptr(), fout + pad, off.data_ptr(), rows, E, fin, fout)
        check(L, L.msr_experts_forward(op[0], op[1], w.data_ptr(), y, *op[4:], stream()))
        check(L, L.msr_experts_dgrad(op[2], op[3], w.data_ptr(), dx, *op[4:], stream()))
        check(L, L.msr_experts_wgrad(dw, *op, stream()))
        check(L, L.msr_experts_wgrad_sr_accum(acc, *op, 9, 0, 1, None, stream()))
        for buffer, view in outs:
            assert bool(torch.isfinite(view).all())
            assert bool((buffer[:64] == 7.0).all()) and bool((buffer[64 + view.numel():] == 7.0).all())
