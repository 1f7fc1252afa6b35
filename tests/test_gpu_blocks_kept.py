"""What a backward pass of the residual-block operators reads is looked at
before the launch: parameters whose data was replaced since the forward pass
and saved-tensor hooks that give back other tensors are errors, or work."""

from __future__ import annotations

import pytest
import torch

from rollfast_amd import autograd as ag
from rollfast_amd import blocks

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


REPLACED = {"cpu": lambda t: t.cpu(), "shorter": lambda t: t[..., :24].clone(),
            "longer": lambda t: torch.cat((t, t), -1), "strided": lambda t: torch.cat((t, t), -1)[..., ::2]}


@pytest.mark.parametrize("how", REPLACED)
@pytest.mark.parametrize("which", ["weight", "bias", "gate", "next_weight", "next_bias"])
def test_replaced_parameters(which, how):
    x, u = rand(8, 48), rand(8, 48, seed=1)
    v = {n: torch.nn.Parameter(rand(8, 48, seed=2) if n == "gate" else rand(48, seed=2))
         for n in ("weight", "bias", "gate", "next_weight", "next_bias")}
    out, y, saved = blocks.postnorm_residual(x, u, **v, norm="layer", next_norm="layer")
    before = blocks.postnorm_residual_grad(x, u, saved)
    old = v[which].data
    v[which].data = REPLACED[how](old)
    with pytest.raises(ValueError, match="do not fit together"):
        blocks.postnorm_residual_grad(x, u, saved)
    v[which].data = old
    for a, b in zip(before, blocks.postnorm_residual_grad(x, u, saved)):
        assert torch.equal(a, b)


def test_replaced_weight_of_a_prenorm():
    x, w = rand(8, 48), torch.nn.Parameter(rand(48, seed=1))
    _, saved = blocks.prenorm(x, w)
    w.data = w.data.cpu()
    with pytest.raises(ValueError, match="do not fit together"):
        blocks.prenorm_grad(x, saved)


def block(x, u, w, save):
    y = ag.prenorm(x, w, save=save)
    h = ag.gated_activation(y, u, save=save)
    out, y = ag.postnorm_residual(x, h, w, gate=u[0], next_norm="rms", save=save)
    return (out * u).sum() + (y * x).sum()


@pytest.mark.parametrize("save", ["int8", "input"])
def test_saved_tensors_on_the_host(save):
    """A hook that moves what was kept to the host and back changes nothing."""
    x, u, w = rand(9, 40).requires_grad_(True), rand(9, 40, seed=1).requires_grad_(True), rand(40, seed=2).requires_grad_(True)
    ref = torch.autograd.grad(block(x, u, w, save), [x, u, w])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (t.device, t.cpu()), lambda s: s[1].to(s[0])):
        loss = block(x, u, w, save)
    for a, b in zip(ref, torch.autograd.grad(loss, [x, u, w])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("form", ["prenorm", "gated", "postnorm"])
@pytest.mark.parametrize("save", ["int8", "input"])
@pytest.mark.parametrize("how", ["cpu", "narrow", "short"])
def test_hooks_that_give_back_other_tensors(form, save, how):
    x, u = rand(9, 40).requires_grad_(True), rand(9, 40, seed=1).requires_grad_(True)
    other = {"cpu": lambda t: t.cpu(), "narrow": lambda t: t.to(torch.float16 if t.is_floating_point() else torch.bool),
             "short": lambda t: t.flatten()[: t.numel() // 2].clone()}[how]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
        loss = {"prenorm": lambda: ag.prenorm(x, save=save), "gated": lambda: ag.gated_activation(x, u, save=save),
                "postnorm": lambda: ag.postnorm_residual(x, u, next_norm="rms", save=save)[1]}[form]().sum()
        with pytest.raises((ValueError, NotImplementedError)):
            loss.backward()
