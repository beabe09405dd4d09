"""Distil a decoder with binary MLPs from its float teacher.

    python examples/distill.py [--steps 200] [--vocab 8192] [--one-pass]

The teacher is a small GPT-shaped decoder over a vocabulary with common and
rare tokens; the student is a fresh one whose MLPs are converted to binary layers.
It learns from the teacher's 32 likeliest tokens at each position, with the mass
that they leave as one more outcome:

    teacher -> nn.token_logprobs(top=32) -> nn.distillation_loss -> backward
            -> AdamW on what is continuous, QSTEOptimizer on the coordinates

``--one-pass`` takes loss and gradient from ``nn.distillation_loss_and_grad``
instead, which reads the logits once.  Before and after, both models score the
same tokens (drawn from the teacher, so its mean log probability is about
minus its entropy) with ``nn.token_logprobs``.  The data is synthetic.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import qste_amd as qste  # noqa: E402


class Block(nn.Module):
    def __init__(self, d: int, heads: int):
        super().__init__()
        self.heads = heads
        self.ln1, self.ln2 = nn.LayerNorm(d), nn.LayerNorm(d)
        self.qkv, self.proj = nn.Linear(d, 3 * d), nn.Linear(d, d)
        self.mlp = nn.Sequential(nn.Linear(d, 4 * d), nn.GELU(approximate="tanh"), nn.Linear(4 * d, d))

    def forward(self, x):
        b, t, d = x.shape
        q, k, v = self.qkv(self.ln1(x)).view(b, t, 3, self.heads, d // self.heads).permute(2, 0, 3, 1, 4)
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        x = x + self.proj(y.transpose(1, 2).reshape(b, t, d))
        return x + self.mlp(self.ln2(x))


class Decoder(nn.Module):
    def __init__(self, vocab: int, d: int, layers: int, heads: int, context: int):
        super().__init__()
        self.tokens, self.places = nn.Embedding(vocab, d), nn.Embedding(context, d)
        self.blocks = nn.ModuleList(Block(d, heads) for _ in range(layers))
        self.norm, self.head = nn.LayerNorm(d), nn.Linear(d, vocab)

    def forward(self, ids):
        x = self.tokens(ids) + self.places.weight[: ids.shape[1]]
        for block in self.blocks:
            x = block(x)
        return self.head(self.norm(x))


def scored(model, ids, targets, context):
    """Mean log probability and entropy of the targets; positions marked -100 do not count."""

    with torch.no_grad(), context:
        s = qste.nn.token_logprobs(model(ids), targets)
    count = (targets >= 0).sum()
    return float(s.logprobs.sum() / count), float(s.entropy.sum() / count)


def main(steps: int = 200, vocab: int = 8192, d: int = 256, layers: int = 4, batch: int = 8, seq: int = 128,
         top: int = 32, one_pass: bool = False, seed: int = 0, verbose: bool = True) -> dict:
    device = torch.device("cuda")
    torch.manual_seed(seed)
    teacher = Decoder(vocab, d, layers, d // 64, seq).to(device)
    with torch.no_grad():
        # an untrained head is nearly flat: give it something to teach, common tokens before all
        teacher.head.weight.mul_(2.0)
        teacher.head.bias.copy_(-1.2 * torch.arange(1, vocab + 1, device=device).float().log())
    student = Decoder(vocab, d, layers, d // 64, seq)
    qste.convert(student, include=["blocks.*.mlp.0", "blocks.*.mlp.2"])
    student.to(device)
    adam = torch.optim.AdamW(qste.continuous_parameters(student), lr=3e-3)
    coords = qste.QSTEOptimizer(student)
    autocast = torch.autocast("cuda", dtype=torch.bfloat16)
    draw = torch.Generator(device=device).manual_seed(seed + 1)

    def batch_of():
        ids = torch.randint(vocab, (batch, seq), generator=draw, device=device)
        ends = torch.randint(seq // 2, seq + 1, (batch, 1), generator=draw, device=device)
        return ids, torch.arange(seq, device=device) < ends  # the last positions of a sequence are padding

    ids, live = batch_of()
    with torch.no_grad(), autocast:
        p = torch.softmax(teacher(ids).float(), -1).view(-1, vocab)
    targets = torch.where(live, torch.multinomial(p, 1, generator=draw).view(batch, seq), -100)
    result = {"teacher": scored(teacher, ids, targets, autocast), "before": scored(student, ids, targets, autocast),
              "losses": []}
    for step in range(steps):
        x, there = batch_of()
        marks = torch.where(there, x, -1)  # a negative token: not scored by the teacher, no entry for the student
        with torch.no_grad(), autocast:
            target = qste.nn.token_logprobs(teacher(x), marks, top=top)
        with autocast:
            logits = student(x)
        if one_pass:
            losses, grad = qste.nn.distillation_loss_and_grad(logits.detach(), target.top_tokens, target.top_logprobs,
                                                              loss_grad=there / there.sum(), tail=True)
            logits.backward(grad)
            loss = losses.sum() / there.sum()
        else:
            losses = qste.nn.distillation_loss(logits, target.top_tokens, target.top_logprobs, tail=True)
            loss = losses.sum() / there.sum()
            loss.backward()
        adam.step()
        adam.zero_grad(set_to_none=True)
        coords.step()
        if step % 20 == 0 or step == steps - 1:
            result["losses"].append(float(loss.detach()))
            if verbose:
                print(f"step {step:4d}  loss {result['losses'][-1]:.4f}", flush=True)
    result["after"] = scored(student, ids, targets, autocast)
    if verbose:
        for name in ("teacher", "before", "after"):
            print(f"{name:8s} log probability {result[name][0]:8.4f}  entropy {result[name][1]:7.4f}")
    return result


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--vocab", type=int, default=8192)
    parser.add_argument("--one-pass", action="store_true")
    args = parser.parse_args()
    main(steps=args.steps, vocab=args.vocab, one_pass=args.one_pass)
