"""Trains a small mixture-of-experts language model with this package's operators on one GPU.

A byte of text predicts the next one through an embedding, two mixture-of-experts blocks (a
router's top 2 of 8 experts for every token) and a head, all bf16.  Each step runs ``SREmbedding``, then per block

    LayerNorm -> router (torch) -> order_tokens -> dispatch_tokens -> SRExperts -> GELU -> SRExperts -> combine_tokens

with the router's ``balance_loss``, and ``SRHead``'s loss, forward and backward over a few micro-batches, whose gradients
``TritonSRAccumulator``, ``SREmbedding``, ``SRExperts`` and ``SRHead`` accumulate with stochastic rounding; ``clip_grad_norm_`` cuts their global norm;
``TritonMuonSRWithAuxAdam`` steps the experts' matrices with Muon and the rest with AdamW.

    python examples/moe_train.py [--steps 200] [--micro 4] [--tokens 4096]
"""
from __future__ import annotations

import argparse
import glob
import os
import sys
import sysconfig

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from muon_sr_amd import (LayerNorm, SREmbedding, SRExperts, SRHead, TritonMuonSRWithAuxAdam,  # noqa: E402
                         TritonSRAccumulator, balance_loss, clip_grad_norm_, combine_tokens, dispatch_tokens, order_tokens)

BF16 = torch.bfloat16


class MoE(nn.Module):
    """y[t] = sum over the chosen experts e of t: weight[t, e] * down_e(gelu(up_e(x[t])))."""

    def __init__(self, d, hidden, experts, k, device):
        super().__init__()
        self.experts, self.k = experts, k
        self.router = nn.Linear(d, experts, bias=False, device=device, dtype=BF16)
        self.up = SRExperts(experts, d, hidden, device=device)
        self.down = SRExperts(experts, hidden, d, device=device)

    def forward(self, x):
        logits = self.router(x)
        scores = torch.softmax(logits.float(), -1)
        weights, ids = torch.topk(scores, self.k, dim=-1)
        weights = weights / weights.sum(-1, keepdim=True)
        order = order_tokens(ids, self.experts)
        rows = dispatch_tokens(x, order)
        rows = self.down(F.gelu(self.up(rows, order.offsets)), order.offsets)
        return combine_tokens(rows, weights, order), balance_loss(logits, ids)[0]


class Model(nn.Module):
    def __init__(self, d=256, hidden=512, experts=8, k=2, blocks=2, context=4, device="cuda"):
        super().__init__()
        self.context = context
        self.embed = SREmbedding(256, d, device=device)
        self.mix = nn.Linear(context * d, d, bias=False, device=device, dtype=BF16)
        self.norms = nn.ModuleList(LayerNorm(d, device=device, dtype=BF16) for _ in range(blocks))
        self.moe = nn.ModuleList(MoE(d, hidden, experts, k, device) for _ in range(blocks))
        self.head = SRHead(d, 256, device=device)

    def features(self, idx):
        """idx: [tokens, context] bytes -> the head's input [tokens, d] and the balance term."""
        x, balance = self.mix(self.embed(idx).flatten(1)), 0.0
        for norm, moe in zip(self.norms, self.moe):
            y, b = moe(norm(x))
            x, balance = x + y, balance + b
        return x, balance

    def forward(self, idx):
        """Logits [tokens, 256] and the balance term."""
        x, balance = self.features(idx)
        return self.head(x), balance

    def loss(self, idx, target):
        """The mean cross entropy and the balance term, without the logits in memory."""
        x, balance = self.features(idx)
        return self.head.loss(x, target), balance


def param_groups(model):
    muon = [p for m in model.moe for p in (m.up.weight, m.down.weight)]
    ids = {id(p) for p in muon}
    rest = [p for p in model.parameters() if id(p) not in ids]
    return [dict(params=muon, lr=0.01, momentum=0.95, weight_decay=0.01, use_muon=True),
            dict(params=rest, lr=2e-3, betas=(0.9, 0.95), eps=1e-10, weight_decay=0.0, use_muon=False)]


def corpus(folder=None, limit=4 << 20):
    """The text of a folder's Python files (default: the running interpreter's standard library), as bytes."""
    folder, text = folder or sysconfig.get_paths()["stdlib"], b""
    for name in sorted(glob.glob(os.path.join(folder, "*.py"))):
        with open(name, "rb") as f:
            text += f.read()
        if len(text) >= limit:
            break
    if len(text) < 1 << 16:
        raise RuntimeError(f"{folder} has only {len(text)} bytes of Python files to train on; 65536 are the least")
    return torch.frombuffer(bytearray(text[:limit]), dtype=torch.uint8).long()


def train(steps=200, micro=4, tokens=4096, max_norm=0.3, seed=0, report=None):
    """The mean loss and the gradient norm (before clipping) of every step."""
    torch.manual_seed(seed)
    model = Model()
    opt = TritonMuonSRWithAuxAdam(param_groups(model), batch_ns=True)
    TritonSRAccumulator.assign_hooks(model)
    data, c = corpus().cuda(), model.context
    gen = torch.Generator(device="cuda").manual_seed(seed)
    losses, norms = [], []
    for step in range(steps):
        total = 0.0
        for _ in range(micro):
            at = torch.randint(0, data.numel() - c, (tokens,), generator=gen, device="cuda")
            window = data[at[:, None] + torch.arange(c + 1, device="cuda")]
            loss, balance = model.loss(window[:, :c], window[:, c])
            ((loss + 0.01 * balance) / micro).backward()
            total = total + loss.detach() / micro
        TritonSRAccumulator.reassign_grad_buffer(model)
        norms.append(clip_grad_norm_(model.parameters(), max_norm))
        opt.step()
        opt.zero_grad(set_to_none=True)
        losses.append(total)
        if report and (step + 1) % report == 0:
            print(f"step {step + 1:4d}  loss {total.item():.4f}  gradient norm {norms[-1].item():.3f}", flush=True)
    return torch.stack(losses).tolist(), torch.stack(norms).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--micro", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=4096)
    a = ap.parse_args()
    train(a.steps, a.micro, a.tokens, report=20)
