"""Timed cases of the operators at a language model's ends and between its blocks: the head's product with its
cross entropy, the embedding, layer norm, and the router's balance loss, with their gradients.

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
import random

import numpy as np
import torch

own = False

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-5
IGNORED = -100


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a few tokens through the smallest model's head, 512 words of width 256, forward and backward (latency)
        dict(name="head_7_512x256", kind="head", rows=7, vocab=512, d=256, ignored=0.0, reduction="mean", accum=False,
             backward=True),
        # a micro-batch of the small GPT: 32 x 128 tokens, 16384 words of width 384
        dict(name="head_4096_16384x384", kind="head", rows=4096, vocab=16384, d=384, ignored=0.0, reduction="mean",
             accum=False, backward=True),
        # an evaluation with a loss per token: odd counts of tokens and words
        dict(name="head_eval_2047_50257x1024", kind="head", rows=2047, vocab=50257, d=1024, ignored=0.1,
             reduction="none", accum=False, backward=False),
        # the 24-layer model of width 2048 with 32000 words, its gradient added to the accumulator, a padded batch
        dict(name="head_accum_8191_32000x2048", kind="head", rows=8191, vocab=32000, d=2048, ignored=0.1,
             reduction="mean", accum=True, backward=True),
        # Llama-3-8B's head: 128256 words of width 4096
        dict(name="head_8192_128256x4096", kind="head", rows=8192, vocab=128256, d=4096, ignored=0.0,
             reduction="mean", accum=False, backward=True),
        # the smallest model's embedding (latency)
        dict(name="embed_61_512x256", kind="embed", tokens=61, vocab=512, d=256, dtype="bf16", scale=1.0, padding=False,
             accum=False),
        # the 24-layer model's embedding: the gradient of an odd number of tokens added to the accumulator
        dict(name="embed_accum_16383_32000x2048", kind="embed", tokens=16383, vocab=32000, d=2048, dtype="bf16",
             scale=45.25483399593904, padding=True, accum=True),
        # Llama-3-8B's embedding with a whole gradient: 16384 tokens
        dict(name="embed_16384_128256x4096", kind="embed", tokens=16384, vocab=128256, d=4096, dtype="bf16", scale=1.0,
             padding=False, accum=False),
        # the small GPT's norms, 17 of them in a pass of its model: 4096 rows of 384 (latency)
        dict(name="norm_4096x384", kind="norm", rows=4096, d=384, dtype="bf16", wdtype="bf16", bias=True),
        # a large batch of width 4096
        dict(name="norm_32768x4096", kind="norm", rows=32768, d=4096, dtype="bf16", wdtype="bf16", bias=True),
        # a router of 64 experts over an ordinary micro-batch, two choices per token (latency)
        dict(name="balance_8192x64", kind="balance", tokens=8192, experts=64, k=2, dtype="bf16", dropped=0.0, masked=0.0),
        # many tokens and experts, a padded batch, some slots dropped
        dict(name="balance_131071x256", kind="balance", tokens=131071, experts=256, k=8, dtype="f32", dropped=0.05,
             masked=0.1),
    ]


MOST_PRODUCT = 8192 * 128256 * 4096      # rows x words x width of the largest head
MOST_LOGITS = 8192 * 128256
MOST_WEIGHT = 128256 * 4096
MOST_SEEDED = 32000 * 4096               # words x width of an accumulator (the plain form's noise takes 8 bytes and more a word)
MOST_NORM = 32768 * 4096
MOST_SCORES = 131072 * 256


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, step):
    """Log-uniform in [lo, hi]: half of them multiples of `step`, the others as they come."""
    v = _log(rng, lo, hi)
    return max(step, v // step * step) if rng.random() < 0.5 else v


def draw(rng):
    kind = rng.choice(["head", "head", "embed", "embed", "norm", "norm", "balance"])
    if kind == "head":
        while True:
            c = dict(kind=kind, rows=_size(rng, 1, 16384, 128), vocab=_size(rng, 17, 131072, 128),
                     d=8 * _log(rng, 2, 1024), ignored=rng.choice([0.0, 0.1, 0.5]),
                     reduction=rng.choice(["mean", "mean", "sum", "none"]), accum=rng.random() < 0.3,
                     backward=rng.random() < 0.8)
            c["accum"] = c["accum"] and c["backward"]
            weight = c["vocab"] * c["d"]
            if c["rows"] * weight <= MOST_PRODUCT and c["rows"] * c["vocab"] <= MOST_LOGITS and \
                    weight <= (MOST_SEEDED if c["accum"] else MOST_WEIGHT):
                return c
    if kind == "embed":
        while True:
            accum = rng.random() < 0.4
            c = dict(kind=kind, tokens=_size(rng, 1, 65536, 64), vocab=_size(rng, 17, 131072, 64),
                     d=8 * _log(rng, 1, 1024) if accum else _size(rng, 5, 8192, 64),
                     dtype="bf16" if accum else rng.choice(["bf16", "bf16", "f32"]),
                     scale=rng.choice([1.0, 1.0, 22.627416997969522]), padding=rng.random() < 0.3, accum=accum)
            size = 2 if c["dtype"] == "f32" else 1
            if c["vocab"] * c["d"] * size <= (MOST_SEEDED if accum else MOST_WEIGHT) and \
                    c["tokens"] * c["d"] * size <= 16384 * 4096:
                return c
    if kind == "norm":
        while True:
            c = dict(kind=kind, rows=_size(rng, 1, 131072, 64), d=_size(rng, 5, 16384, 64),
                     dtype=rng.choice(["bf16", "bf16", "f32"]), wdtype=rng.choice(["bf16", "f32"]),
                     bias=rng.random() < 0.7)
            if c["rows"] * c["d"] * (2 if c["dtype"] == "f32" else 1) <= MOST_NORM:
                return c
    while True:
        k = rng.choice([1, 2, 2, 3, 4, 8])
        c = dict(kind=kind, tokens=_size(rng, 1, 131072, 64), experts=_size(rng, max(2, k), 512, 8), k=k,
                 dtype=rng.choice(["bf16", "f32"]), dropped=rng.choice([0.0, 0.05]), masked=rng.choice([0.0, 0.0, 0.1]))
        if c["tokens"] * c["experts"] <= MOST_SCORES:
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, std, gen, dtype=BF16):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype).mul_(std)


def _rand(shape, gen):
    return torch.rand(shape, generator=gen, device=DEV)


def _type(name):
    return BF16 if name == "bf16" else F32


def _words(n, vocab, gen):
    """Word v with a probability that falls as 1 / (v + 1), as the words of a text sorted by frequency."""
    return (torch.exp(_rand((n,), gen).double() * math.log(vocab + 1)).long() - 1).clamp_(0, vocab - 1)


def _prepare_head(case, gen):
    """Logits of standard deviation 3; rows that know their word from not at all to nearly surely; rows to
    ignore in runs of 50."""
    n, vocab, d = case["rows"], case["vocab"], case["d"]
    w = _randn((vocab, d), 3.0 / math.sqrt(d), gen)
    target = _words(n, vocab, gen)
    x = _randn((n, d), 1.0, gen)
    x += (_rand((n, 1), gen) * 2.5).to(BF16) * w[target]
    if case["ignored"]:
        run = _rand((n // 50 + 1,), gen) < case["ignored"]
        target.masked_fill_(run.repeat_interleave(50)[:n], IGNORED)
    s = dict(case=case, x=x.requires_grad_(case["backward"]), w=torch.nn.Parameter(w, requires_grad=case["backward"]),
             target=target, dloss=_rand((n,) if case["reduction"] == "none" else (), gen).add_(0.25))
    if case["accum"]:
        s["seed"] = int(torch.randint(0, 1 << 32, (1,), generator=gen, device=DEV))
        s["w"].acc_grad = _randn((vocab, d), 1e-4, gen)
        if own:
            from muon_sr_amd import SRHead
            s["head"] = SRHead(d, vocab, device="meta", dtype=BF16)
            s["head"].weight = s["w"]
    return s


def _prepare_embed(case, gen):
    n, vocab, d, dt = case["tokens"], case["vocab"], case["d"], _type(case["dtype"])
    ids = _words(n, vocab, gen)
    s = dict(case=case, ids=ids, pad=vocab // 3 if case["padding"] else None, dy=_randn((n, d), 1e-2, gen, dt))
    if case["padding"]:                        # a tenth of the batch is padding
        ids.masked_fill_(_rand((n,), gen) < 0.1, s["pad"])
    s["w"] = torch.nn.Parameter(_randn((vocab, d), 0.02, gen, dt))
    if case["accum"]:
        s["seed"] = int(torch.randint(0, 1 << 32, (1,), generator=gen, device=DEV))
        s["w"].acc_grad = _randn((vocab, d), 1e-2, gen)
    return s


def _prepare_norm(case, gen):
    """Rows of different size and columns of different mean, weights around one."""
    n, d, dt, wt = case["rows"], case["d"], _type(case["dtype"]), _type(case["wdtype"])
    x = _randn((n, d), 1.0, gen, dt)
    x.mul_(_rand((n, 1), gen).add_(0.2).to(dt)).add_(_randn((d,), 0.5, gen, dt))
    return dict(case=case, x=x.requires_grad_(True), w=_randn((d,), 0.1, gen, wt).add_(1.0).requires_grad_(True),
                b=_randn((d,), 0.1, gen, wt).requires_grad_(True) if case["bias"] else None,
                dy=_randn((n, d), 1e-2, gen, dt))


def _prepare_balance(case, gen):
    """A router's logits, some experts wanted more than others, and the choice by them."""
    n, e, k = case["tokens"], case["experts"], case["k"]
    logits = (_randn((n, e), 1.0, gen, F32) + _randn((e,), 0.7, gen, F32)).to(_type(case["dtype"]))
    ids = torch.topk(logits.float(), k, dim=1).indices
    if case["dropped"]:
        ids = ids.masked_fill(_rand((n, k), gen) < case["dropped"], -1)
    return dict(case=case, logits=logits.requires_grad_(True), ids=ids, dloss=_rand((), gen).add_(0.01),
                mask=_rand((n,), gen) >= case["masked"] if case["masked"] else None)


def prepare(case, seed):
    gen = _gen(seed)
    with torch.no_grad():
        return {"head": _prepare_head, "embed": _prepare_embed, "norm": _prepare_norm,
                "balance": _prepare_balance}[case["kind"]](case, gen)


# ---------------------------------------------------------------------------
# one pass: the package's calls
# ---------------------------------------------------------------------------

def _own_head(s):
    from muon_sr_amd import linear_cross_entropy
    case = s["case"]
    if case["accum"]:
        random.seed(s["seed"])
        loss = s["head"].loss(s["x"], s["target"], reduction=case["reduction"])
        dx, = torch.autograd.grad(loss, (s["x"],), s["dloss"])
        return dict(loss=loss, dx=dx, acc=s["w"].acc_grad)
    loss = linear_cross_entropy(s["x"], s["w"], s["target"], reduction=case["reduction"])
    if not case["backward"]:
        return dict(loss=loss)
    dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]), s["dloss"])
    return dict(loss=loss, dx=dx, dw=dw)


def _own_embed(s):
    from muon_sr_amd import embedding, embedding_grad_sr_accum
    case = s["case"]
    y = embedding(s["ids"], s["w"], padding_idx=s["pad"], scale=case["scale"])
    if case["accum"]:
        embedding_grad_sr_accum(s["w"], s["ids"], s["dy"], padding_idx=s["pad"], scale=case["scale"], seed=s["seed"])
        return dict(y=y, acc=s["w"].acc_grad)
    dw, = torch.autograd.grad(y, (s["w"],), s["dy"])
    return dict(y=y, dw=dw)


def _own_norm(s):
    from muon_sr_amd import layer_norm
    y = layer_norm(s["x"], s["w"], s["b"], EPS)
    leaves = [t for t in (s["x"], s["w"], s["b"]) if t is not None]
    return [y, *torch.autograd.grad(y, leaves, s["dy"])]


def _own_balance(s):
    from muon_sr_amd import balance_loss
    loss, counts = balance_loss(s["logits"], s["ids"], mask=s["mask"])
    dlogits, = torch.autograd.grad(loss, (s["logits"],), s["dloss"])
    return dict(loss=loss, counts=counts, dlogits=dlogits)


# ---------------------------------------------------------------------------
# one pass: the plain forms
# ---------------------------------------------------------------------------

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


def _accumulate(acc, dw, seed):
    """acc <- SR(acc + dw): 16 noise bits added below the bits that are kept."""
    bits = (acc.float() + dw.float()).view(torch.int32).long() + _philox16(seed, acc.numel()).view(acc.shape)
    return acc.copy_((bits & 0xFFFF0000).to(torch.int32).view(F32))


def _plain_head(s):
    case, x, w, target = s["case"], s["x"].detach(), s["w"].detach(), s["target"]
    kept = target != IGNORED
    word = torch.where(kept, target, 0)
    p = x.float() @ w.float().t()
    top = p.max(1).values
    picked = p.gather(1, word[:, None])[:, 0]
    lse = top + (p - top[:, None]).exp_().sum(1).log()
    loss = torch.where(kept, lse - picked, 0)
    count = kept.sum().clamp(min=1)
    if case["reduction"] == "sum":
        loss = loss.sum()
    elif case["reduction"] == "mean":
        loss = loss.sum() / count
    if not case["backward"]:
        return dict(loss=loss)
    g = torch.where(kept, s["dloss"] / count if case["reduction"] == "mean" else s["dloss"], 0)
    p.sub_(lse[:, None]).exp_().mul_(g[:, None])
    p[torch.arange(len(word), device=DEV), word] -= g
    dx = (p @ w.float()).to(BF16)
    dw = (p.t() @ x.float()).to(BF16)
    if not case["accum"]:
        return dict(loss=loss, dx=dx, dw=dw)
    random.seed(s["seed"])
    return dict(loss=loss, dx=dx, acc=_accumulate(s["w"].acc_grad, dw, random.getrandbits(32)))


def _plain_embed(s):
    case, w, ids = s["case"], s["w"].detach(), s["ids"]
    y = (w[ids].float() * case["scale"]).to(w.dtype)
    dy = s["dy"].float()
    if s["pad"] is not None:
        dy = torch.where((ids != s["pad"])[:, None], dy, 0)
    dw = torch.zeros(w.shape, dtype=F32, device=DEV).index_add_(0, ids, dy)
    dw = (dw * case["scale"]).to(w.dtype)
    return dict(y=y, acc=_accumulate(s["w"].acc_grad, dw, s["seed"])) if case["accum"] else dict(y=y, dw=dw)


def _plain_norm(s):
    x, w, dy = s["x"].detach().float(), s["w"].detach().float(), s["dy"].float()
    x = x - x.mean(1, keepdim=True)
    r = (x.square().mean(1, keepdim=True) + EPS).rsqrt()
    h = x * r
    y = h * w
    if s["b"] is not None:
        y = y + s["b"].detach().float()
    q = dy * w
    dx = (q - q.mean(1, keepdim=True) - h * (q * h).mean(1, keepdim=True)) * r
    wt = s["w"].dtype
    out = [y.to(s["x"].dtype), dx.to(s["x"].dtype), (dy * h).sum(0).to(wt)]
    return out + [dy.sum(0).to(wt)] if s["b"] is not None else out


def _plain_balance(s):
    case, ids = s["case"], s["ids"]
    e, mask = case["experts"], s["mask"]
    p = s["logits"].detach().float()
    p = (p - p.max(1, keepdim=True).values).exp()
    p = p / p.sum(1, keepdim=True)
    there = (ids >= 0) & (ids < e)
    if mask is not None:
        p, there = torch.where(mask[:, None], p, 0), there & mask[:, None]
    n = mask.sum().clamp(min=1) if mask is not None else len(p)
    counts = torch.zeros(e, dtype=torch.int64, device=DEV).index_add_(0, ids.clamp(0, e - 1).flatten(), there.long().flatten())
    f = counts.float() / (n * case["k"])
    loss = (f * p.sum(0)).sum() * e / n
    d = p * (f - (p * f).sum(1, keepdim=True)) * (s["dloss"] * e / n)
    return dict(loss=loss, counts=counts.int(), dlogits=d.to(s["logits"].dtype))


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"head": _own_head, "embed": _own_embed, "norm": _own_norm, "balance": _own_balance}[kind](state)
    return {"head": _plain_head, "embed": _plain_embed, "norm": _plain_norm, "balance": _plain_balance}[kind](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _distinct(n, vocab):
    """Words that n tokens hit, on average."""
    p = np.diff(np.log(np.arange(1, vocab + 2))) / math.log(vocab + 1)
    return float((1.0 - (1.0 - p) ** n).sum())


def work(case):
    if case["kind"] == "head":
        n, weight, d = round(case["rows"] * (1 - case["ignored"])), case["vocab"] * case["d"], case["d"]
        if not case["backward"]:
            return {"bytes": 2 * (n * d + weight) + 8 * case["rows"], "flops": 2 * n * weight}
        return {"bytes": 2 * (n * d + weight) + 8 * case["rows"] + 2 * case["rows"] * d + (4 if case["accum"] else 2) * weight,
                "flops": 6 * n * weight}
    if case["kind"] == "embed":
        n, d, size = case["tokens"], case["d"], 2 if case["dtype"] == "bf16" else 4
        rows = _distinct(n, case["vocab"])
        written = 2 * rows if case["accum"] else case["vocab"]        # of the accumulator: read and written
        return {"bytes": round(8 * n + size * d * (rows + 2 * n + written)), "flops": 2 * n * d}
    if case["kind"] == "norm":
        n, size = case["rows"] * case["d"], 2 if case["dtype"] == "bf16" else 4
        vectors = 2 * case["d"] * (2 if case["wdtype"] == "bf16" else 4) * (2 if case["bias"] else 1)
        return {"bytes": 4 * n * size + vectors, "flops": 18 * n}
    n = case["tokens"] * case["experts"]
    return {"bytes": 2 * n * (2 if case["dtype"] == "bf16" else 4) + 8 * case["tokens"] * case["k"], "flops": 12 * n}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_head(s):
    """1024 rows at a time.  An accumulator's value is the one that stochastic rounding has on average: the
    unrounded sum."""
    case, target = s["case"], s["target"]
    w = s["w"].detach().double()
    kept = (target != IGNORED).nonzero().flatten()
    n = len(target)
    loss = torch.zeros(n, dtype=torch.float64, device=DEV)
    dx = torch.zeros((n, case["d"]), dtype=torch.float64, device=DEV)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=DEV) if case["backward"] else None
    scale = 1.0 / max(1, len(kept)) if case["reduction"] == "mean" else 1.0
    for rows in kept.split(1024):
        x, t = s["x"].detach()[rows].double(), target[rows]
        z = x @ w.t()
        lse = torch.logsumexp(z, 1)
        at = torch.arange(len(rows), device=DEV)
        loss[rows] = lse - z[at, t]
        if case["backward"]:
            g = (s["dloss"].double() * scale).expand(n)[rows].unsqueeze(1)
            z = torch.exp(z - lse.unsqueeze(1))
            z[at, t] -= 1.0
            z *= g
            dx[rows] = z @ w
            dw.addmm_(z.t(), x)
    if case["reduction"] != "none":
        loss = loss.sum() * scale
    if not case["backward"]:
        return dict(loss=loss)
    if case["accum"]:
        return dict(loss=loss, dx=dx, acc=dw + s["w"].acc_grad.double())
    return dict(loss=loss, dx=dx, dw=dw)


def _exact_embed(s):
    """Rows sorted by word; each word's sum is the difference of two sums of all before it, column block by
    column block."""
    case, ids, w = s["case"], s["ids"], s["w"].detach()
    y = w[ids].double() * case["scale"]
    keep = (ids != s["pad"]).nonzero().flatten() if s["pad"] is not None else torch.arange(len(ids), device=DEV)
    word, order = torch.sort(ids[keep])
    dw = s["w"].acc_grad.double() if case["accum"] else torch.zeros(w.shape, dtype=torch.float64, device=DEV)
    if len(keep):
        hit, many = torch.unique_consecutive(word, return_counts=True)
        end = many.cumsum(0)
        for c in range(0, case["d"], 1024):
            run = s["dy"][keep[order], c:c + 1024].double().cumsum(0)[end - 1]
            run[1:] = run[1:] - run[:-1].clone()
            dw[hit, c:c + 1024] += run * case["scale"]
    return dict(y=y, acc=dw) if case["accum"] else dict(y=y, dw=dw)


def _exact_norm(s):
    """8192 rows at a time; dx from the projection form of the gradient."""
    n, d = s["x"].shape
    w = s["w"].detach().double()
    y, dx = (torch.empty((n, d), dtype=torch.float64, device=DEV) for _ in range(2))
    dw, db = (torch.zeros(d, dtype=torch.float64, device=DEV) for _ in range(2))
    for i in range(0, n, 8192):
        x, dy = s["x"].detach()[i:i + 8192].double(), s["dy"][i:i + 8192].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        sd = torch.sqrt(var + EPS)
        h = (x - mean) / sd
        y[i:i + 8192] = h * w + (s["b"].detach().double() if s["b"] is not None else 0.0)
        q = dy * w
        dx[i:i + 8192] = (q - (q.sum(1, keepdim=True) + h * (q * h).sum(1, keepdim=True)) / d) / sd
        dw += (dy * h).sum(0)
        db += dy.sum(0)
    return [y, dx, dw] + ([db] if s["b"] is not None else [])


def _exact_balance(s):
    """Counts from numpy; the gradient through the softmax's Jacobian."""
    case = s["case"]
    e, n = case["experts"], case["tokens"]
    mask = s["mask"].cpu().numpy() if s["mask"] is not None else np.ones(n, dtype=bool)
    ids = s["ids"].cpu().numpy()[mask]
    counts = np.bincount(ids[(ids >= 0) & (ids < e)], minlength=e)
    n = max(1, int(mask.sum()))
    share = torch.from_numpy(counts / (n * case["k"])).to(DEV)
    p = torch.softmax(s["logits"].detach().double(), 1)
    p[torch.from_numpy(~mask).to(DEV)] = 0.0
    loss = e * torch.dot(share, p.sum(0) / n)
    slope = share * (e / n * float(s["dloss"]))
    return dict(loss=loss, counts=None, dlogits=p * slope - p * (p @ slope).unsqueeze(1))


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"head": _exact_head, "embed": _exact_embed, "norm": _exact_norm,
                "balance": _exact_balance}[case["kind"]](s)
