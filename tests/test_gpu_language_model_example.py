"""The operators of a training step together, as the language model's example has
them: its gradients against a plain model in 64 bits, its optimizer's updates
against their definitions, and that it runs."""

from __future__ import annotations

import importlib.util
import math
import os

import numpy as np
import pytest
import torch

import rollfast_amd as rf
from tests.test_gpu_muon8 import step
from tests.test_gpu_orthogonalize import BOUND, exact

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_language_model", os.path.join(ROOT, "examples", "train_language_model.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


SIZES = dict(vocab=301, hidden=96, ffn=136, layers=2)


def setting(example, dtype, seed=3):
    params = example.init(SIZES["vocab"], SIZES["hidden"], SIZES["ffn"], SIZES["layers"], dtype, seed)
    tokens, targets = next(example.batches(SIZES["vocab"], 3, 37, 5, seed))
    return params, tokens, targets


def plain(params, tokens, targets, z_loss=1e-4):
    """The model in 64 bits, from its definition."""
    def norm(x, w):
        return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w

    blocks = [params[k] for k in sorted(params) if k.startswith("block")]
    x = params["embed"][tokens]
    y = norm(x, blocks[0]["norm_in"])
    for i, p in enumerate(blocks):
        gate, up = (y @ p["gate_up"].t()).chunk(2, -1)
        branch = (gate * torch.sigmoid(gate) * up) @ p["down"].t()
        x = x + p["gate"] * norm(branch, p["norm_out"])
        y = norm(x, params["norm_head"] if i + 1 == len(blocks) else blocks[i + 1]["norm_in"])
    logits = y @ params["head"].t()
    lse = torch.logsumexp(logits, -1)
    losses = lse - logits.gather(-1, targets.clamp(min=0)[..., None])[..., 0] + z_loss * lse * lse
    return losses[targets >= 0].mean()


def tree_map(f, *trees):
    return {k: tree_map(f, *(t[k] for t in trees)) if isinstance(trees[0][k], dict) else f(*(t[k] for t in trees)) for k in trees[0]}


def flat(tree, name=""):
    return {n: v for k, x in tree.items() for n, v in (flat(x, f"{name}{k}.") if isinstance(x, dict) else {f"{name}{k}": x}).items()}


def test_gradients(example):
    """In f32 with whole inputs.  The longest sums have 301 terms, and a gradient has
    passed through at most 25 operations (5 a block forward and backward, the head, the
    loss, the norms), each off by at most 301 half steps of 2^-24 of its terms' size:
    25 * 301 * 2^-24 = 4.5e-4, which twofold stands for terms that cancel."""
    params, tokens, targets = setting(example, torch.float32)
    value, grads = example.loss_and_grads(params, tokens, targets, save="input")
    wide = tree_map(lambda p: p.detach().double().cpu().requires_grad_(True), params)
    ref = plain(wide, tokens.cpu(), targets.cpu())
    ref.backward()
    assert abs(value.item() - ref.item()) < 4.5e-4 * ref.item()  # the loss is of its logits' size or more: log(301) = 5.7
    got = flat(grads)
    for name, leaf in flat(wide).items():
        off = (got[name].double().cpu() - leaf.grad).norm().item()
        assert off < 9e-4 * leaf.grad.norm().item(), (name, off, leaf.grad.norm().item())


def test_gradients_by_differences(example):
    """Along the gradient's own direction in each leaf: with h = 1e-3 |p| the second
    difference of the plain loss in 64 bits is off by h^2, 1e-6 times third derivatives
    of the order of one over |p|^2; the bound leaves 100 times that and the gradient's own."""
    params, tokens, targets = setting(example, torch.float32, seed=5)
    _, grads = example.loss_and_grads(params, tokens, targets, save="input")
    wide = flat(tree_map(lambda p: p.detach().double().cpu(), params))
    tokens, targets = tokens.cpu(), targets.cpu()

    def at(name, change):
        tree = {}
        for n, v in wide.items():
            parts, here = n.split("."), tree
            for k in parts[:-1]:
                here = here.setdefault(k, {})
            here[parts[-1]] = v + change if n == name else v
        return plain(tree, tokens, targets).item()

    for name, g in flat(grads).items():
        g = g.double().cpu()
        along = g / g.norm()
        h = 1e-3 * wide[name].norm().item()
        slope = (at(name, h * along) - at(name, -h * along)) / (2 * h)
        assert abs(slope - g.norm().item()) < 9e-4 * g.norm().item() + 1e-4 * abs(slope), (name, slope, g.norm().item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step(example, dtype):
    """Each leaf's update from the gradients: the matrices' orthogonalised momentum,
    the rest as adamw8 alone gives them."""
    params, tokens, targets = setting(example, dtype)
    tx = example.optimizer(params)
    state = tx.init(params)
    alone = rf.adamw8(learning_rate=3e-3, weight_decay=0.01)
    names = [n for n in flat(params) if not n.endswith(("gate_up", "down"))]
    alone_state = alone.init({n: flat(params)[n] for n in names})
    momentum = {}
    for _ in range(2):
        _, grads = example.loss_and_grads(params, tokens, targets)
        kept = {n: m for n, m in momentum.items()}
        updates, state = tx.update(grads, state, params)
        p, g, u = flat(params), flat(grads), flat(updates)
        want, alone_state = alone.update({n: g[n] for n in names}, alone_state, {n: p[n] for n in names})
        for n in names:
            assert torch.equal(u[n], want[n]), n
        stored = flat(state.inner_states["matrix"].inner_state.mu)
        for n in p:
            if n in names:
                continue
            old = kept.get(n, np.zeros(tuple(p[n].shape), np.float32))
            _, direction = step(old, g[n].float().cpu().numpy(), 0.95, True)
            r, c = p[n].shape
            s = math.sqrt(max(1.0, r / c))
            ref = -0.02 * (s * exact(torch.from_numpy(direction).cuda()) + 0.01 * p[n].double())
            size = 0.02 * (s * math.sqrt(min(r, c)) * 1.2 + 0.01 * p[n].double().norm().item())
            assert (u[n].double() - ref).norm().item() < BOUND[dtype] * size, n
            momentum[n] = rf.dequantize_blocks(stored[n]).cpu().numpy()
        params = rf.apply_updates(params, updates, stochastic=False)
        assert all(x.dtype == p[n].dtype and torch.isfinite(x).all() for n, x in flat(params).items())


@pytest.mark.parametrize("save", ["int8", "input"])
def test_example_runs(example, save):
    losses, params = example.train(4, save=save)
    assert len(losses) == 4 and all(math.isfinite(x) for x in losses)
    assert all(torch.isfinite(p).all() for p in flat(params).values())
