"""Trains a small language model of gated feed-forward blocks, with a loss that
writes no logits and 8-bit state for both of its optimizers.

The blocks' matrices are updated by ``muon8`` (orthogonalised momentum, the
momentum in 8-bit blocks), the embedding, the head and the norms by ``adamw8``;
``multi_transform`` has them as one transformation.  The head and the loss are
``linear_cross_entropy``: the loss and the gradients of the head and of its input
in one pass, in which the exponentials of a piece of the tokens are all that is held
by vocabulary.  Tokens of a sequence's prompt are
ignored by the loss.

    python examples/train_language_model.py [--steps 50] [--save int8|input]

prints the loss of a synthetic next-token task.
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

IGNORED = -100


def init(vocab, hidden, ffn, layers, dtype, seed=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def matrix(outs, cols):
        return (torch.randn(outs, cols, generator=gen, device="cuda") / math.sqrt(cols)).to(dtype)

    def ones(value=1.0):
        return torch.full((hidden,), value, device="cuda")

    params = {"embed": matrix(vocab, hidden), "head": matrix(vocab, hidden), "norm_head": ones()}
    for i in range(layers):
        params[f"block{i}"] = {"norm_in": ones(), "gate_up": matrix(2 * ffn, hidden), "down": matrix(hidden, ffn),
                               "norm_out": ones(), "gate": ones(1.0 / layers)}
    return params


def optimizer(params, lr=3e-3, matrix_lr=0.02, weight_decay=0.01):
    """``muon8`` for the blocks' matrices, ``adamw8`` for all else."""

    def label(tree):
        return {k: label(v) if isinstance(v, dict) else "matrix" if k in ("gate_up", "down") else "rest" for k, v in tree.items()}

    return rf.multi_transform({"matrix": rf.muon8(matrix_lr, weight_decay=weight_decay),
                               "rest": rf.adamw8(learning_rate=lr, weight_decay=weight_decay)}, label(params))


def loss(params, tokens, targets, save="int8", z_loss=1e-4):
    """The mean loss of the targets that are not ignored.  ``save``: what the
    layers keep of their inputs for the backward pass."""
    kept8 = save == "int8"

    def linear(x, weight, kept):
        return ag.linear(x, weight, checkpoint=kept) if kept8 else torch.nn.functional.linear(x, weight)

    blocks = [params[k] for k in sorted(params) if k.startswith("block")]
    x = torch.nn.functional.embedding(tokens, params["embed"])
    y, kept = ag.prenorm(x, blocks[0]["norm_in"], save=save, checkpoint_output=kept8) if kept8 else \
        (ag.prenorm(x, blocks[0]["norm_in"], save=save), None)
    for i, p in enumerate(blocks):
        last = i + 1 == len(blocks)
        gate_up = linear(y, p["gate_up"], kept)
        h, kept = ag.gated_activation(gate_up, save=save, checkpoint_output=True) if kept8 else \
            (ag.gated_activation(gate_up, save=save), None)
        branch = linear(h, p["down"], kept)
        got = ag.postnorm_residual(x, branch, p["norm_out"], gate=p["gate"], next_norm="rms",
                                   next_weight=params["norm_head"] if last else blocks[i + 1]["norm_in"], save=save,
                                   checkpoint_output=kept8 and not last)  # the loss keeps gradients, not its input
        x, y, kept = got if len(got) == 3 else (*got, None)
    return ag.linear_cross_entropy(y, params["head"], targets, ignore_index=IGNORED, z_loss=z_loss)


def _leaves(tree):
    return [leaf for k in sorted(tree) for leaf in (_leaves(tree[k]) if isinstance(tree[k], dict) else [tree[k]])]


def _like(tree, leaves):
    return {k: _like(tree[k], leaves) if isinstance(tree[k], dict) else next(leaves) for k in sorted(tree)}


def loss_and_grads(params, tokens, targets, save="int8"):
    leaves = _leaves(params)
    for leaf in leaves:
        leaf.requires_grad_(True)
    value = loss(params, tokens, targets, save)
    grads = torch.autograd.grad(value, leaves)
    for leaf in leaves:
        leaf.requires_grad_(False)
    return value.detach(), _like(params, iter(grads))


def batches(vocab, batch, length, prompt, seed):
    """(tokens, targets) without end: each token's successor nine times in ten;
    the first ``prompt`` targets of a sequence are ignored."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    follow = torch.randint(0, vocab, (vocab,), generator=gen, device="cuda")
    while True:
        tokens = torch.randint(0, vocab, (batch, length), generator=gen, device="cuda")
        noise = torch.rand(batch, length, generator=gen, device="cuda") < 0.1
        targets = torch.where(noise, torch.randint(0, vocab, (batch, length), generator=gen, device="cuda"), follow[tokens])
        targets[:, :prompt] = IGNORED
        yield tokens, targets


def train(steps=50, *, vocab=1000, hidden=256, ffn=704, layers=4, batch=16, length=128, prompt=16, dtype=torch.bfloat16,
          save="int8", seed=0):
    """The losses, and the parameters."""
    params = init(vocab, hidden, ffn, layers, dtype, seed)
    tx = optimizer(params)
    state = tx.init(params)
    losses = []
    for step, (tokens, targets) in zip(range(steps), batches(vocab, batch, length, prompt, seed + 1)):
        value, grads = loss_and_grads(params, tokens, targets, save)
        updates, state = tx.update(grads, state, params)
        params = rf.apply_updates(params, updates, stochastic=False)
        losses.append(value)
    return [float(x) for x in losses], params


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--save", choices=("int8", "input"), default="int8")
    args = ap.parse_args()
    losses, _ = train(args.steps, save=args.save)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i:4d}  loss {losses[i]:.4f}")
    print(f"last loss {losses[-1]:.4f}")


if __name__ == "__main__":
    main()
