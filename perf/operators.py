"""Timed cases of the operators around the optimizer step: the global gradient norm with
clipping, tokens sorted by expert and back, and the experts' products with their gradients.

``own`` false: each operator in its plain form, elementary torch operations in 32 bits,
rounded once at the end.  ``own`` true: the package's public calls.

    listed()                the cases that are always measured
    draw(rng)               one more case of the same ranges
    prepare(case, seed)     what a program has before the call, on the GPU
    run(state)              one pass; its outputs
    work(case)              bytes and flops that the pass cannot do without
    exact(case, seed)       the outputs in 64 bits, from the operators' definitions
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
CLIP_EPS = 1e-6


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the smallest model's gradients: 4 matrices of 256 x 256, two vectors, a 512 x 256 embedding (latency)
        dict(name="clip_4x256", kind="clip", shapes="hybrid", d=256, vocab=512, dtype="bf16", norm=2.0),
        # the gradients of the small GPT: 8 layers of width 384, vocabulary 16384, 73 tensors
        dict(name="clip_8L_d384", kind="clip", shapes="model", layers=8, d=384, ffn=1536, vocab=16384, dtype="bf16",
             norm=2.0),
        # fp32 gradients of odd lengths, as views that are not 16-byte aligned, clipped into bf16 ones
        dict(name="clip_odd_fp32", kind="clip", shapes="odd", tensors=12, numel=5000001, dtype="f32", norm=2.0),
        # a large model's accumulation buffers: 24 layers of width 2048, 217 tensors, 1.3 billion elements
        dict(name="clip_24L_d2048", kind="clip", shapes="model", layers=24, d=2048, ffn=5632, vocab=32000,
             dtype="bf16", norm=2.0),
        # a handful of tokens through a layer that is only evaluated (latency)
        dict(name="tokens_7x384", kind="tokens", tokens=7, k=2, experts=8, d=384, dtype="bf16", wdtype="f32",
             dropped=0.0, backward=False),
        # fp32 activations, odd counts, many experts and a tenth of the slots without one
        dict(name="tokens_5003x1400_fp32", kind="tokens", tokens=5003, k=3, experts=160, d=1400, dtype="f32",
             wdtype="f32", dropped=0.1, backward=True),
        # an ordinary micro-batch: 8192 tokens of width 2048, 2 of 64 experts
        dict(name="tokens_8192x2048", kind="tokens", tokens=8192, k=2, experts=64, d=2048, dtype="bf16", wdtype="f32",
             dropped=0.0, backward=True),
        # the largest: 32768 tokens, 8 of 128 experts
        dict(name="tokens_32768x2048", kind="tokens", tokens=32768, k=8, experts=128, d=2048, dtype="bf16",
             wdtype="bf16", dropped=0.0, backward=True),
        # few rows and small experts, forward and backward (latency)
        dict(name="experts_61_8x512x256", kind="experts", rows=61, spare=3, experts=8, fout=512, fin=256, accum=False),
        # the small GPT's MLP as 8 experts, at its batch of 32 x 128 tokens with 2 experts each
        dict(name="experts_8192_8x1536x384", kind="experts", rows=8192, spare=0, experts=8, fout=1536, fin=384,
             accum=False),
        # many experts of width 2048 with uneven, odd counts: the weight gradients' accumulation
        dict(name="experts_accum_16411_64x1024x2048", kind="experts", rows=16411, spare=57, experts=64, fout=1024,
             fin=2048, accum=True),
        # 8 experts of Llama-3-8B's MLP width
        dict(name="experts_8192_8x14336x4096", kind="experts", rows=8192, spare=0, experts=8, fout=14336, fin=4096,
             accum=False),
    ]


MOST_MOVED = 32768 * 8 * 2048              # tokens x k x d of the largest case
MOST_PRODUCT = 8192 * 14336 * 4096         # rows x out x in of the largest case
MOST_WEIGHTS = 8 * 14336 * 4096


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return v + 8 if v == 24 * 128 else v


def _size(rng, lo, hi, step):
    """Log-uniform in [lo, hi]: half of them multiples of `step`, the others as they come."""
    v = _log(rng, lo, hi)
    v = max(step, v // step * step) if rng.random() < 0.5 else v
    return v + step if v == 24 * 128 else v


def draw(rng):
    kind = rng.choice(["clip", "tokens", "experts", "experts"])
    if kind == "clip":
        norm = rng.choice([2.0, 2.0, 2.0, 1.0, math.inf])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        if rng.random() < 0.5:
            return dict(kind=kind, shapes="model", layers=rng.randint(1, 24), d=_size(rng, 128, 2048, 64),
                        ffn=_size(rng, 256, 5632, 64), vocab=_size(rng, 500, 32000, 64), dtype=dtype, norm=norm)
        return dict(kind=kind, shapes="odd", tensors=rng.randint(1, 300), numel=_size(rng, 1, 1 << 24, 8), dtype=dtype,
                    norm=norm)
    if kind == "tokens":
        while True:
            k = rng.choice([1, 2, 2, 3, 4, 6, 8])
            c = dict(kind=kind, tokens=_size(rng, 1, 32768, 64), k=k, experts=_size(rng, max(2, k), 256, 8),
                     d=_size(rng, 24, 8192, 64), dtype=rng.choice(["bf16", "bf16", "f32"]),
                     wdtype=rng.choice(["bf16", "f32"]), dropped=rng.choice([0.0, 0.0, 0.1]),
                     backward=rng.random() < 0.7)
            if c["tokens"] * k * c["d"] * (2 if c["dtype"] == "f32" else 1) <= MOST_MOVED:
                return c
    while True:
        fout, fin = (8 * (_size(rng, 64, 14336, 64) // 8) for _ in range(2))
        c = dict(kind=kind, rows=_size(rng, 1, 32768, 128), spare=rng.choice([0, 0, rng.randint(1, 100)]),
                 experts=_log(rng, 1, 128), fout=fout, fin=fin, accum=rng.random() < 0.4)
        if c["rows"] * fout * fin <= MOST_PRODUCT and c["experts"] * fout * fin <= MOST_WEIGHTS // 2:
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, std, gen, dtype=BF16):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype).mul_(std)


def _type(name):
    return BF16 if name == "bf16" else F32


def _clip_shapes(case):
    d, v = case.get("d"), case.get("vocab")
    if case["shapes"] == "hybrid":
        return [(d, d)] * 4 + [(d,), (d,), (v, d)]
    if case["shapes"] == "model":
        f = case["ffn"]
        return ([(d, d)] * 4 + [(f, d), (f, d), (d, f)] + [(d,), (d,)]) * case["layers"] + [(v, d)]
    return [(max(0, case["numel"] // (i + 1) - i),) for i in range(case["tensors"])]


def _views(shapes, dtype, odd):
    """Views of one flat buffer (zeros), 128-byte aligned or (`odd`) at odd elements."""
    at, offs = 0, []
    for s in shapes:
        offs.append(at + odd)
        at += -(-(math.prod(s) + odd) // 64) * 64
    flat = torch.zeros(max(1, at), dtype=dtype, device=DEV)
    return flat, [flat[o:o + math.prod(s)].view(s) for o, s in zip(offs, shapes)]


def _prepare_clip(case, gen):
    """Gradients whose size differs from tensor to tensor, a bound that cuts them to about a half, and the
    gradients that the step will read."""
    shapes, odd = _clip_shapes(case), case["shapes"] == "odd"
    flat, grads = _views(shapes, _type(case["dtype"]), odd)
    flat.normal_(0.0, 1e-3, generator=gen)
    scales = torch.rand(len(shapes), generator=gen, device=DEV).add_(0.1).tolist()
    for g, s in zip(grads, scales):
        g.mul_(s)
    n = sum(math.prod(s) for s in shapes)
    bound = {1.0: 2e-4 * n, 2.0: 3e-4 * math.sqrt(n), math.inf: 5e-4}[case["norm"]]
    out, outs = _views(shapes, BF16, odd)
    return dict(case=case, grads=grads, max_norm=max(bound, 1e-7), out=out, outs=outs)


def _prepare_tokens(case, gen):
    """A router's choice (some experts wanted more than others), its weights, and the activations and
    gradients on both sides of the experts."""
    T, k, E, d, dt = case["tokens"], case["k"], case["experts"], case["d"], _type(case["dtype"])
    logits = _randn((T, E), 1.0, gen, F32) + _randn((E,), 0.7, gen, F32)
    top, ids = torch.topk(logits, k, dim=1)
    if case["dropped"]:
        ids = ids.masked_fill(torch.rand((T, k), generator=gen, device=DEV) < case["dropped"], -1)
    s = dict(case=case, ids=ids, experts=E, x=_randn((T, d), 1.0, gen, dt), w=torch.softmax(top, 1).to(_type(case["wdtype"])),
             r=_randn((T * k, d), 1.0, gen, dt))
    if case["backward"]:
        s["drows"], s["dy"] = _randn((T * k, d), 1e-3, gen, dt), _randn((T, d), 1e-3, gen, dt)
        for name in ("x", "w", "r"):
            s[name].requires_grad_(True)
    return s


def _prepare_experts(case, gen):
    """Rows sorted by expert, in uneven groups (some empty), with `spare` rows after the last group."""
    E, n = case["experts"], case["rows"]
    share = torch.softmax(_randn((E,), 0.7, gen, F32), 0)
    ids = torch.multinomial(share, n, replacement=True, generator=gen)
    counts = torch.zeros(E, dtype=torch.int64, device=DEV).index_add_(0, ids, torch.ones_like(ids))
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
    offsets[1:] = counts.cumsum(0)
    rows = n + case["spare"]
    s = dict(case=case, offsets=offsets, x=_randn((rows, case["fin"]), 1.0, gen),
             w=torch.nn.Parameter(_randn((E, case["fout"], case["fin"]), 0.02, gen)),
             dy=_randn((rows, case["fout"]), 1e-2, gen))
    if case["accum"]:
        s["seed"] = int(torch.randint(0, 1 << 32, (1,), generator=gen, device=DEV))
        s["w"].acc_grad = _randn((E, case["fout"], case["fin"]), 1e-2, gen)
    else:
        s["x"].requires_grad_(True)
    return s


def prepare(case, seed):
    gen = _gen(seed)
    return {"clip": _prepare_clip, "tokens": _prepare_tokens, "experts": _prepare_experts}[case["kind"]](case, gen)


# ---------------------------------------------------------------------------
# one pass: the package's calls
# ---------------------------------------------------------------------------

def _own_clip(s):
    from muon_sr_amd import clip_grads
    return [clip_grads(s["grads"], s["max_norm"], norm_type=s["case"]["norm"], out=s["outs"]), s["out"]]


def _own_tokens(s):
    from muon_sr_amd import combine_tokens, dispatch_tokens, order_tokens
    order = order_tokens(s["ids"], s["experts"])
    rows = dispatch_tokens(s["x"], order)
    y = combine_tokens(s["r"], s["w"], order)
    out = dict(offsets=order.offsets, position=order.position, source=order.source, rows=rows, y=y)
    if s["case"]["backward"]:
        out["dx"], out["dr"], out["dw"] = torch.autograd.grad((rows, y), (s["x"], s["r"], s["w"]), (s["drows"], s["dy"]))
    return out


def _own_experts(s):
    from muon_sr_amd import expert_linear, experts_wgrad_sr_accum
    if s["case"]["accum"]:
        experts_wgrad_sr_accum(s["w"], s["x"], s["dy"], s["offsets"], seed=s["seed"])
        return dict(acc=s["w"].acc_grad)
    y = expert_linear(s["x"], s["w"], s["offsets"])
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return dict(y=y, dx=dx, dw=dw)


# ---------------------------------------------------------------------------
# one pass: the plain forms
# ---------------------------------------------------------------------------

def _plain_clip(s):
    p = s["case"]["norm"]
    if p == math.inf:
        norm = torch.stack([g.float().abs().max() for g in s["grads"] if g.numel()]).max()
    elif p == 1.0:
        norm = torch.stack([g.float().abs().sum() for g in s["grads"]]).sum()
    else:
        norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    c = (s["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0)
    for g, o in zip(s["grads"], s["outs"]):
        o.copy_(g.float() * c)
    return [norm, s["out"]]


def _plain_tokens(s):
    ids, E, k = s["ids"], s["experts"], s["case"]["k"]
    n = ids.numel()
    at = torch.arange(n, device=DEV)
    key = torch.where((ids >= 0) & (ids < E), ids, E).flatten()
    counts = torch.zeros(E + 1, dtype=torch.int64, device=DEV).index_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([counts.new_zeros(1), counts[:E].cumsum(0)])
    source = torch.sort(key, stable=True).indices
    held = at < offsets[E]                                           # rows with a slot
    position = torch.empty_like(at).index_copy_(0, source, at)
    position = torch.where(key < E, position, -1).view(ids.shape)
    source = torch.where(held, source, -1)
    there = (position >= 0)[:, :, None]
    take = position.clamp(min=0)
    token = source.clamp(min=0) // k
    x, r, w = s["x"].detach(), s["r"].detach(), s["w"].detach().float()
    rows = torch.where(held[:, None], x[token], 0)
    picked = torch.where(there, r.float()[take], 0)
    y = (picked * w[:, :, None]).sum(1).to(x.dtype)
    out = dict(offsets=offsets.int(), position=position.int(), source=source.int(), rows=rows, y=y)
    if s["case"]["backward"]:
        dy = s["dy"].float()
        out["dx"] = torch.where(there, s["drows"].float()[take], 0).sum(1).to(x.dtype)
        out["dr"] = torch.where(held[:, None], dy[token] * w.flatten()[source.clamp(min=0)][:, None], 0).to(r.dtype)
        out["dw"] = (picked * dy[:, None, :]).sum(2).to(s["w"].dtype)
    return out


def _philox16(seed, n):
    """16 noise bits for each of n offsets (n a multiple of 8): Philox4x32-10 of counter offset // 8 under the
    key `seed`, 16 bits per offset (Salmon et al., SC'11)."""
    m32 = 0xFFFFFFFF
    k0, k1 = seed & m32, 0                # a seed of 2^31 and more is a 64-bit integer: high word 0 all the same
    c0 = torch.arange(n // 8, device=DEV, dtype=torch.int64)
    c1, c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0), torch.zeros_like(c0)
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & m32) ^ c1 ^ k0, b & m32, ((a >> 32) & m32) ^ c3 ^ k1, a & m32
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).view(-1)


def _plain_experts(s):
    case, off, E = s["case"], s["offsets"].long(), s["case"]["experts"]
    x, dy, w = s["x"].detach(), s["dy"], s["w"].detach()
    at = torch.arange(x.shape[0], device=DEV)
    cap = max(1, int((off[1:] - off[:-1]).max()))
    held = at < off[E]
    e = torch.searchsorted(off[1:], at, right=True).clamp(max=E - 1)
    slot = torch.where(held, e * cap + at - off[e], E * cap)         # the last one takes the spare rows
    place = lambda v: torch.zeros(E * cap + 1, v.shape[1], dtype=F32, device=DEV).index_copy_(  # noqa: E731
        0, slot, torch.where(held[:, None], v.float(), 0))[:E * cap].view(E, cap, -1)
    back = lambda v: torch.where(held[:, None], v.reshape(E * cap, -1)[slot.clamp(max=E * cap - 1)], 0).to(BF16)  # noqa: E731
    xp, dyp, wf = place(x), place(dy), w.float()
    dw = torch.bmm(dyp.transpose(1, 2).contiguous(), xp).to(BF16)
    if case["accum"]:
        acc = s["w"].acc_grad
        bits = (acc.float() + dw.float()).view(torch.int32).long() + _philox16(s["seed"], acc.numel()).view(acc.shape)
        acc.copy_((bits & 0xFFFF0000).to(torch.int32).view(F32))
        return dict(acc=acc)
    y = torch.bmm(xp, wf.transpose(1, 2).contiguous())
    return dict(y=back(y), dx=back(torch.bmm(dyp, wf)), dw=dw)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"clip": _own_clip, "tokens": _own_tokens, "experts": _own_experts}[kind](state)
    return {"clip": _plain_clip, "tokens": _plain_tokens, "experts": _plain_experts}[kind](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["kind"] == "clip":
        n = sum(math.prod(s) for s in _clip_shapes(case))
        return {"bytes": n * ((2 if case["dtype"] == "bf16" else 4) + 2) + 4, "flops": 3 * n}
    if case["kind"] == "tokens":
        T, k, d = case["tokens"], case["k"], case["d"]
        size, wsize, n = 2 if case["dtype"] == "bf16" else 4, 2 if case["wdtype"] == "bf16" else 4, T * k
        full = round(n * (1 - case["dropped"]))            # slots with an expert
        b = n * (8 + 4 + 4 + wsize) + 4 * (case["experts"] + 1)
        b += size * d * (T + n) + size * d * (full + T)    # x -> rows, r -> y
        f = 2 * full * d
        if case["backward"]:
            b += size * d * (full + T)                     # drows -> dx
            b += size * d * (T + n) + n * wsize            # dy -> dr, dw (r and the weights are read above)
            f += full * d + full * d + 2 * full * d
        return {"bytes": b, "flops": f}
    E, o, i, n = case["experts"], case["fout"], case["fin"], case["rows"]
    total = n + case["spare"]
    if case["accum"]:
        return {"bytes": 2 * n * (o + i) + 4 * E * o * i, "flops": 2 * n * o * i}
    return {"bytes": 2 * n * (o + i) + 2 * total * (o + i) + 4 * E * o * i, "flops": 6 * n * o * i}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_clip(s):
    p, total = s["case"]["norm"], 0.0
    for g in s["grads"]:
        if g.numel():
            a = g.double().abs()
            total = max(total, a.max().item()) if p == math.inf else total + (a ** p).sum().item()
    norm = total if p == math.inf else total ** (1.0 / p)
    c = min(1.0, s["max_norm"] / (norm + CLIP_EPS))
    odd = int(s["case"]["shapes"] == "odd")
    out, at = torch.zeros(s["out"].numel(), dtype=torch.float64, device=DEV), 0
    for g in s["grads"]:
        out[at + odd:at + odd + g.numel()] = g.double().flatten() * c
        at += -(-(g.numel() + odd) // 64) * 64
    return [np.float64(norm), out]


def _exact_tokens(s):
    """Slot by slot in numpy for the order, then one of a token's k slots at a time."""
    ids, E = s["ids"].cpu().numpy(), s["experts"]
    T, k = ids.shape
    flat = ids.reshape(-1)
    lists = [np.nonzero(flat == e)[0] for e in range(E)]
    src = np.concatenate(lists)
    pos = np.full(T * k, -1, dtype=np.int64)
    pos[src] = np.arange(len(src))
    tok, slot = torch.from_numpy(src // k).to(DEV), torch.from_numpy(src).to(DEV)
    pos = torch.from_numpy(pos.reshape(T, k)).to(DEV)
    x, r, w = s["x"].detach().double(), s["r"].detach().double(), s["w"].detach().double()
    n = len(src)
    rows = torch.zeros_like(r)
    rows[:n] = x[tok]
    y = torch.zeros_like(x)
    bw = s["case"]["backward"]
    if bw:
        dy, drows = s["dy"].double(), s["drows"].double()
        dx, dr, dw = torch.zeros_like(x), torch.zeros_like(r), torch.zeros_like(w)
        dr[:n] = dy[tok] * w.reshape(-1)[slot].unsqueeze(1)
    for j in range(k):
        t = torch.nonzero(pos[:, j] >= 0).flatten()
        at = pos[t, j]
        y[t] += r[at] * w[t, j].unsqueeze(1)
        if bw:
            dx[t] += drows[at]
            dw[t, j] = (r[at] * dy[t]).sum(1)
    out = dict(offsets=None, position=None, source=None, rows=rows, y=y)
    return dict(out, dx=dx, dr=dr, dw=dw) if bw else out


def _exact_experts(s):
    """One expert after the other.  An accumulator's value is the one that stochastic rounding has on
    average: the unrounded sum."""
    off = s["offsets"].tolist()
    x, dy, w = s["x"].detach(), s["dy"], s["w"].detach()
    accum = s["case"]["accum"]
    y = torch.zeros(dy.shape, dtype=torch.float64, device=DEV)
    dx = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    dw = s["w"].acc_grad.double() if accum else torch.zeros(w.shape, dtype=torch.float64, device=DEV)
    for e in range(len(off) - 1):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        xe, de = x[lo:hi].double(), dy[lo:hi].double()
        dw[e] += de.t().contiguous() @ xe
        if not accum:
            we = w[e].double()
            y[lo:hi] = xe @ we.t().contiguous()
            dx[lo:hi] = de @ we
    return dict(acc=dw) if accum else dict(y=y, dx=dx, dw=dw)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"clip": _exact_clip, "tokens": _exact_tokens, "experts": _exact_experts}[case["kind"]](s)
