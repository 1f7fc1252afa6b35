"""Trains a small stack of gated feed-forward blocks with 8-bit optimizer state
and 8-bit saved activations.

Each block is: the norm before it, a gated feed-forward layer (one product for
gate and up, the gated activation, one product down), and the norm after it
with a learned gate per channel and the residual sum; the end of a block and
the norm before the next one are one pass.  Linear layers keep their inputs as
checkpoints that the norms and the gated activation made in the same pass.  The
optimizer is ``adamw8_step``.

    python examples/train_gated_blocks.py [--steps 50] [--save int8|input]

prints the loss of a synthetic next-token task and the bytes that the backward
pass of a step keeps.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import rollfast_amd as rf  # noqa: E402
from rollfast_amd import autograd as ag  # noqa: E402


def init(vocab, hidden, ffn, layers, dtype, seed=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def matrix(outs, cols):
        return (torch.randn(outs, cols, generator=gen, device="cuda") / math.sqrt(cols)).to(dtype)

    def ones(value=1.0):
        return torch.full((hidden,), value, device="cuda")

    params = {"embed": matrix(vocab, hidden), "head": matrix(vocab, hidden)}
    for i in range(layers):
        params[f"block{i}"] = {"norm_in": ones(), "gate_up": matrix(2 * ffn, hidden), "down": matrix(hidden, ffn),
                               "norm_out": ones(), "gate": ones(1.0 / layers)}
    params["norm_head"] = ones()
    return params


def forward(params, tokens, save="int8"):
    """Logits of the next token."""
    blocks = [params[k] for k in sorted(params) if k.startswith("block")]
    x = torch.nn.functional.embedding(tokens, params["embed"])
    y, kept = ag.prenorm(x, blocks[0]["norm_in"], save=save, checkpoint_output=True)
    for i, p in enumerate(blocks):
        last = i + 1 == len(blocks)
        gate_up = ag.linear(y, p["gate_up"], checkpoint=kept)
        h, kept = ag.gated_activation(gate_up, save=save, checkpoint_output=True)
        branch = ag.linear(h, p["down"], checkpoint=kept)
        x, y, kept = ag.postnorm_residual(x, branch, p["norm_out"], gate=p["gate"], next_norm="rms",
                                          next_weight=params["norm_head"] if last else blocks[i + 1]["norm_in"],
                                          save=save, checkpoint_output=True)
    return ag.linear(y, params["head"], checkpoint=kept)


def _leaves(tree):
    return [leaf for k in sorted(tree) for leaf in (_leaves(tree[k]) if isinstance(tree[k], dict) else [tree[k]])]


def _like(tree, leaves):
    return {k: _like(tree[k], leaves) if isinstance(tree[k], dict) else next(leaves) for k in sorted(tree)}


def train(steps=50, *, vocab=512, hidden=256, ffn=704, layers=4, batch=16, length=128, dtype=torch.bfloat16, save="int8",
          lr=3e-3, seed=0):
    """(losses, bytes kept for the backward pass of a step)."""
    params = init(vocab, hidden, ffn, layers, dtype, seed)
    tx = rf.adamw8(learning_rate=lr, weight_decay=0.01)
    state = tx.init(params)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed + 1)
    follow = torch.randint(0, vocab, (vocab,), generator=gen, device="cuda")  # each token's successor, most of the time
    losses, kept = [], 0
    for step in range(steps):
        tokens = torch.randint(0, vocab, (batch, length), generator=gen, device="cuda")
        noise = torch.rand(batch, length, generator=gen, device="cuda") < 0.1
        target = torch.where(noise, torch.randint(0, vocab, (batch, length), generator=gen, device="cuda"), follow[tokens])
        leaves = _leaves(params)
        for leaf in leaves:
            leaf.requires_grad_(True)
        before = torch.cuda.memory_allocated()
        logits = forward(params, tokens, save)
        loss = torch.nn.functional.cross_entropy(logits.view(-1, vocab).float(), target.view(-1))
        kept = torch.cuda.memory_allocated() - before
        grads = torch.autograd.grad(loss, leaves)
        losses.append(loss.detach())
        del logits, loss
        for leaf in leaves:
            leaf.requires_grad_(False)
        params, state = rf.adamw8_step(tx, params, _like(params, iter(grads)), state, stochastic=False)
    return [float(x) for x in losses], kept


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--save", choices=("int8", "input"), default="int8")
    args = ap.parse_args()
    losses, kept = train(args.steps, save=args.save)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i:4d}  loss {losses[i]:.4f}")
    print(f"last loss {losses[-1]:.4f}; kept for the backward pass: {kept / 2 ** 20:.1f} MiB")


if __name__ == "__main__":
    main()
