"""The two ends of a training step of a language model, as timed cases.

Where the step's gradients begin and where its matrices' updates end:

- ``loss``: the softmax cross entropy of ``hidden @ weight.T`` over a large
  vocabulary, a number per token, for evaluation (``linear_cross_entropy``);
- ``loss_grad``: the same with the gradients of ``hidden`` and ``weight``
  (``linear_cross_entropy_grad``);
- ``orthogonalize``: matrices with their singular values brought near one by
  Newton-Schulz products (``orthogonalize``);
- ``muon``: an optimizer step's updates from gradients, with the momentum in
  8-bit blocks and orthogonalised matrices (``muon8``).

Definitions.  A token's loss is ``lse - logit[target] + z_loss * lse^2`` with
lse the log of the sum of its logits' exponentials; tokens whose target is
``IGNORE`` have a loss of zero and no part in the gradients, which are those of
``sum(dloss * loss)``.  Newton-Schulz: ``X = G / (|G| + EPS)`` with the
Frobenius norm, then STEPS times ``X = a X + (b A + c A^2) X`` with A = X X^T.
Momentum: ``m = beta m + (1 - beta) g``, stored as the nearest of 256 codes and a
scale (the largest magnitude) per block of 2048 elements; the direction is
``beta m + (1 - beta) g`` with m before it is stored, its update
``-lr (sqrt(max(1, rows / cols)) X + decay p)``.

Sizes: hidden 4096, feed-forward 11008 and vocabulary 32000 (the 7B model of the
optimizer's benchmark), 768 and 50257 (its small language model); odd ones.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
MOMENTUM, RATE, DECAY, QUANT = 0.95, 0.02, 0.1, 2048

ATTENTION, UP, DOWN = (4096, 4096), (11008, 4096), (4096, 11008)


def listed():
    return [
        # scoring one token of an answer: the vocabulary's weights are read once
        {"name": "loss_token", "kind": "loss", "tokens": 1, "vocab": 32000, "hidden": 4096, "dtype": "bf16",
         "masked": 0.0, "z_loss": 0.0},
        # evaluating a small language model on eight sequences of 1024
        {"name": "loss_eval_small_lm", "kind": "loss", "tokens": 8192, "vocab": 50257, "hidden": 768, "dtype": "bf16",
         "masked": 0.0, "z_loss": 0.0},
        # a short fine-tuning example in f16, half of it the prompt
        {"name": "loss_grad_short_f16", "kind": "loss_grad", "tokens": 67, "vocab": 32000, "hidden": 4096,
         "dtype": "f16", "masked": 0.5, "z_loss": 0.0},
        # training a small language model
        {"name": "loss_grad_small_lm", "kind": "loss_grad", "tokens": 8192, "vocab": 50257, "hidden": 768,
         "dtype": "bf16", "masked": 0.0, "z_loss": 0.0},
        # training a 7B model on eight sequences of 2048, a tenth of them padding
        {"name": "loss_grad_llama", "kind": "loss_grad", "tokens": 16384, "vocab": 32000, "hidden": 4096,
         "dtype": "bf16", "masked": 0.1, "z_loss": 1e-4},
        # a large vocabulary of odd size: more logits than are held at once
        {"name": "loss_grad_wide_vocab", "kind": "loss_grad", "tokens": 6001, "vocab": 131101, "hidden": 2048,
         "dtype": "bf16", "masked": 0.0, "z_loss": 0.0},
        # a small f32 model of odd sizes
        {"name": "loss_grad_odd_f32", "kind": "loss_grad", "tokens": 1031, "vocab": 5003, "hidden": 517,
         "dtype": "f32", "masked": 0.3, "z_loss": 1e-4},
        # one small matrix: latency
        {"name": "orthogonalize_small", "kind": "orthogonalize", "shapes": "256x768", "dtype": "bf16"},
        # f32 matrices of odd sizes, wide, tall and square
        {"name": "orthogonalize_odd_f32", "kind": "orthogonalize", "shapes": "517x301 301x1283 641x641 97x1001",
         "dtype": "f32"},
        # the attention and one feed-forward matrix of a 7B layer
        {"name": "orthogonalize_llama", "kind": "orthogonalize", "shapes": "4096x4096 4096x11008", "dtype": "bf16"},
        # all attention matrices of a small language model
        {"name": "muon_small_lm", "kind": "muon", "shapes": " ".join(["2304x768", "768x768"] * 12), "dtype": "bf16"},
        # a whole 7B layer
        {"name": "muon_llama_layer", "kind": "muon",
         "shapes": " ".join(["4096x4096"] * 4 + ["11008x4096"] * 2 + ["4096x11008"]), "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Half of them multiples of 64, half of them any number."""
    n = _log_int(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def _schulz_flops(rows, cols):
    """Of STEPS steps, each symmetric product counted once: n^2 m + n^3 + 2 n^2 m."""
    n, m = min(rows, cols), max(rows, cols)
    return STEPS * (3 * n * n * m + n * n * n)


def draw(rng):
    kind = rng.choice(["loss", "loss_grad", "loss_grad", "orthogonalize", "orthogonalize", "muon"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    if kind in ("loss", "loss_grad"):
        tokens, vocab, hidden = _log_int(rng, 1, 16384), _size(rng, 100, 150000), _size(rng, 40, 5000)
        most = 16384 * 32000 * 4096 // {"bf16": 1, "f16": 1, "f32": 4}[dtype]
        while tokens * vocab * hidden > most or tokens * vocab > 8e8:
            tokens = max(1, tokens * 2 // 3)
        return {"kind": kind, "tokens": tokens, "vocab": vocab, "hidden": hidden, "dtype": dtype,
                "masked": rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.9), 2)]),
                "z_loss": rng.choice([0.0, 0.0, 1e-4])}
    shapes, flops, most = [], 0, 2.0e12 if dtype == "bf16" else 4.0e11
    for _ in range(rng.choice([1, 1, 2, rng.randint(3, 40)])):
        shape = (_size(rng, 24, 8192), _size(rng, 24, 8192))
        if flops + _schulz_flops(*shape) <= most:
            shapes.append(shape)
            flops += _schulz_flops(*shape)
    shapes = shapes or [(_size(rng, 24, 1024), _size(rng, 24, 1024))]
    return {"kind": kind, "shapes": " ".join(f"{r}x{c}" for r, c in shapes), "dtype": dtype}


def _shapes(case):
    return [tuple(map(int, s.split("x"))) for s in case["shapes"].split()]


def _kept(case):
    return case["tokens"] - int(case["tokens"] * case["masked"])


# ------------------------------------------------------------ the inputs ---
def _gradient(gen, rows, cols):
    """A matrix' gradient: a few strong directions over a floor of noise."""
    rank = max(1, min(rows, cols, 64) // 2)
    left = torch.randn(rows, rank, generator=gen, device="cuda")
    right = torch.randn(rank, cols, generator=gen, device="cuda")
    left *= torch.exp(-torch.arange(rank, device="cuda") / 8.0)
    return (left @ right).add_(torch.randn(rows, cols, generator=gen, device="cuda"), alpha=0.3).mul_(1e-3)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] in ("loss", "loss_grad"):
        tokens, vocab, hidden = case["tokens"], case["vocab"], case["hidden"]
        weight = torch.randn(vocab, hidden, generator=gen, device="cuda") * 0.02
        targets = torch.randint(vocab, (tokens,), generator=gen, device="cuda")
        # rows as a last norm leaves them, which know something of the target
        rows = torch.randn(tokens, hidden, generator=gen, device="cuda")
        knows = torch.rand(tokens, 1, generator=gen, device="cuda") * 10.0  # the target's logit above the others'
        rows += knows * weight[targets] / weight[targets].square().sum(1, keepdim=True)
        targets[torch.randperm(tokens, generator=gen, device="cuda")[_kept(case):]] = IGNORE
        s["hidden"], s["weight"], s["targets"] = rows.to(dtype), weight.to(dtype), targets
        # a mean over the tokens that count
        s["dloss"] = torch.full((tokens,), 1.0 / _kept(case), device="cuda")
        return s
    s["grads"] = [_gradient(gen, r, c).to(dtype) for r, c in _shapes(case)]
    if case["kind"] == "muon":
        s["params"] = [(torch.randn(r, c, generator=gen, device="cuda") * 0.02).to(dtype) for r, c in _shapes(case)]
        # momentum of the steps before: like the gradient, in its codes
        s["moments"] = [_encode(_gradient(gen, r, c) * 0.5) for r, c in _shapes(case)]
    return s


def run(state):
    return (_run_own if own else _run_plain)(state)


# ---------------------------------------------- the framework's operators ---
def _run_own(s):
    import rollfast_amd as rf

    case = s["case"]
    if case["kind"] == "loss":
        return rf.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], ignore_index=IGNORE,
                                       z_loss=case["z_loss"])
    if case["kind"] == "loss_grad":
        got = rf.linear_cross_entropy_grad(s["hidden"], s["weight"], s["targets"], s["dloss"], ignore_index=IGNORE,
                                           z_loss=case["z_loss"])
        return got.loss, got.hidden, got.weight
    if case["kind"] == "orthogonalize":
        return rf.orthogonalize(s["grads"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    if "tx" not in s:
        s["tx"] = rf.muon8(RATE, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY, steps=STEPS,
                           coefficients=COEFFICIENTS, eps=EPS, block_size=QUANT, min_size=0)
        mu = [rf.QuantizedBlocks(values=codes, scales=scales, shape=shape, size=math.prod(shape), block_size=QUANT)
              for (codes, scales), shape in zip(s["moments"], _shapes(case))]
        s["state"] = s["tx"].init(s["params"])
        s["state"] = s["state"]._replace(mu=mu)
    updates, s["state"] = s["tx"].update(s["grads"], s["state"], s["params"])
    return updates, [rf.dequantize_blocks(q) for q in s["state"].mu]


# ------------------------------------------------------- the plain forms ---
def _run_plain(s):
    case, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    if case["kind"] in ("loss", "loss_grad"):
        return _plain_loss(s, case, dtype)
    if case["kind"] == "orthogonalize":
        return [_plain_schulz(g.float()).to(dtype) for g in s["grads"]]
    got = [_plain_muon(g, m, p) for g, m, p in zip(s["grads"], s["moments"], s["params"])]
    for (codes, scales), (_, (new_codes, new_scales), _) in zip(s["moments"], got):
        codes.copy_(new_codes)
        scales.copy_(new_scales)
    return [update for update, _, _ in got], [stored for _, _, stored in got]


def _plain_loss(s, case, dtype):
    hidden, weight, targets = s["hidden"].float(), s["weight"].float(), s["targets"]
    counts = targets != IGNORE
    at = torch.where(counts, targets, 0)[:, None]
    logits = hidden @ weight.t()
    top = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at) - top
    scaled = logits.sub_(top).exp_()
    total = scaled.sum(1, keepdim=True)
    lse = top + total.log()
    loss = torch.where(counts, (total.log() - picked + case["z_loss"] * lse * lse)[:, 0], 0.0)
    if case["kind"] == "loss":
        return loss
    dloss = torch.where(counts, s["dloss"], 0.0)[:, None]
    spread = 1 + 2 * case["z_loss"] * lse
    dlogits = scaled.mul_(spread / total * dloss)
    # at the target: probability - 1 without cancellation
    below = torch.expm1(picked - total.log()) + (spread - 1) * (picked - total.log()).exp()
    dlogits.scatter_(1, at, below * dloss)
    return loss, (dlogits @ weight).to(dtype), (dlogits.t() @ hidden).to(dtype)


def _plain_schulz(g):
    a, b, c = COEFFICIENTS
    x = g.t() if g.shape[0] > g.shape[1] else g
    x = x / (x.norm() + EPS)
    for _ in range(STEPS):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if g.shape[0] > g.shape[1] else x


def _book():
    """The dynamic 8-bit map: seven decades of evenly spaced bin means, 0 and 1."""
    edges = [np.linspace(0.1, 1.0, (1 << i) + 1) for i in range(7)]
    means = np.concatenate([(e[:-1] + e[1:]) / 2.0 * 10.0 ** (i - 6) for i, e in enumerate(edges)])
    return torch.tensor(np.sort(np.concatenate([means, -means, [0.0, 1.0]])), dtype=torch.float32, device="cuda")


def _encode(m):
    """(codes [blocks, QUANT], scales [blocks]) of m in f32: largest magnitudes, nearest codes, ties to the lower."""
    blocks = torch.nn.functional.pad(m.reshape(-1), (0, -m.numel() % QUANT)).view(-1, QUANT)
    scales = blocks.abs().amax(1)
    scales = torch.where(scales > 0, scales, 1.0)
    book, x = _book(), blocks / scales[:, None]
    upper = torch.bucketize(x, book, out_int32=True).clamp_(1, 255)  # book[upper - 1] < x <= book[upper] within it
    nearer = (book[upper] - x).abs() < (x - book[upper - 1]).abs()
    return torch.where(nearer, upper, upper - 1).to(torch.uint8), scales


def _decode(codes, scales, shape):
    return (_book()[codes.int()] * scales[:, None]).view(-1)[: math.prod(shape)].view(shape)


def _plain_muon(grad, moment, param):
    g, shape = grad.float(), grad.shape
    m = MOMENTUM * _decode(*moment, shape) + (1 - MOMENTUM) * g
    x = _plain_schulz(MOMENTUM * m + (1 - MOMENTUM) * g)
    update = -RATE * (math.sqrt(max(1.0, shape[0] / shape[1])) * x + DECAY * param.float())
    kept = _encode(m)
    return update.to(grad.dtype), kept, _decode(*kept, shape)


# ------------------------------------------------------- in 64 bits ---------
def _schulz64(g):
    a, b, c = COEFFICIENTS
    x = g.double()
    tall = x.size(0) > x.size(1)
    x = x / (x.pow(2).sum().sqrt() + EPS)
    for _ in range(STEPS):
        if tall:
            k = torch.matmul(x.t().contiguous(), x)
            x = a * x + torch.matmul(x, b * k + c * torch.matmul(k, k))
        else:
            k = torch.matmul(x, x.t().contiguous())
            x = a * x + torch.matmul(b * k + c * torch.matmul(k, k), x)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("loss", "loss_grad"):
        return _loss64(s, case)
    if case["kind"] == "orthogonalize":
        return [_schulz64(g) for g in s["grads"]]
    updates = []
    for g, (codes, scales), p in zip(s["grads"], s["moments"], s["params"]):
        old = _book().double()[codes.long()].mul_(scales.double().unsqueeze(1)).flatten()[: g.numel()].reshape(g.shape)
        new = MOMENTUM * old + (1 - MOMENTUM) * g.double()
        x = _schulz64(MOMENTUM * new + (1 - MOMENTUM) * g.double())
        updates.append(-RATE * (max(1.0, g.size(0) / g.size(1)) ** 0.5 * x + DECAY * p.double()))
    return updates, [None] * len(updates)  # what is stored goes to the nearest code of an f32 value


def _loss64(s, case):
    """By runs of tokens: 64-bit logits of all would not fit beside them."""
    weight = s["weight"].double()
    step = max(1, 2 ** 28 // case["vocab"])
    loss = torch.zeros(case["tokens"], dtype=torch.float64, device="cuda")
    dh = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(weight)
    for t in range(0, case["tokens"], step):
        rows = torch.nonzero(s["targets"][t: t + step] != IGNORE)[:, 0] + t
        h, target = s["hidden"][rows].double(), s["targets"][rows]
        z = torch.matmul(h, weight.t().contiguous())
        lse = torch.logsumexp(z, 1)
        mine = torch.arange(len(rows), device="cuda")
        loss[rows] = lse - z[mine, target] + case["z_loss"] * lse ** 2
        if case["kind"] == "loss_grad":
            p = torch.exp(z - lse[:, None]) * (1 + 2 * case["z_loss"] * lse)[:, None]
            p[mine, target] -= 1.0
            p *= s["dloss"][rows].double()[:, None]
            dh[rows] = torch.matmul(p, weight)
            dw += torch.matmul(p.t().contiguous(), h)
    return loss if case["kind"] == "loss" else (loss, dh, dw)


def work(case):
    """Bytes: every input read and every output written once.  Operations: the
    products of the tokens that count (logits, and for the gradients two of the
    same size); of Newton-Schulz, symmetric products once."""
    b = BYTES[case["dtype"]]
    if case["kind"] in ("loss", "loss_grad"):
        rows, vocab, hidden = _kept(case), case["vocab"], case["hidden"]
        once = (case["tokens"] * hidden + vocab * hidden) * b + case["tokens"] * 12
        grad = case["kind"] == "loss_grad"
        return {"bytes": 2 * once if grad else once, "flops": (6 if grad else 2) * rows * vocab * hidden}
    elements = sum(r * c for r, c in _shapes(case))
    flops = sum(_schulz_flops(r, c) for r, c in _shapes(case))
    # muon: gradient, parameter, update and the codes each way
    return {"bytes": elements * (2 * b if case["kind"] == "orthogonalize" else 3 * b + 2), "flops": flops}
