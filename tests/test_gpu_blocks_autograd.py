"""The differentiable forms of the residual-block operators in a training
program: autocast, gradients that do not come, outputs dropped without a
backward pass, main gradients that something else has kept."""

from __future__ import annotations

import gc

import pytest
import torch

from rollfast_amd import autograd as ag
from rollfast_amd import blocks

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rand(*shape, dtype=F32, seed=0, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


@pytest.mark.parametrize("save", ["int8", "input"])
def test_outputs_dropped_without_a_backward_pass(save):
    """What a forward pass keeps goes with its outputs."""
    x, u = rand(512, 2048).requires_grad_(True), rand(512, 2048, seed=1).requires_grad_(True)

    def forward():
        y, _ = ag.prenorm(x, save=save, checkpoint_output=True)
        out, y2, _ = ag.postnorm_residual(x, u, gate=u[0], next_norm="rms", save=save, checkpoint_output=True)
        h, _ = ag.gated_activation(y2, u, save=save, checkpoint_output=True)
        return (ag.linear(h, u[:64]) + out.sum() + y.sum()).sum()

    forward()
    gc.collect()
    before = torch.cuda.memory_allocated()
    for _ in range(3):
        forward()
    gc.collect()
    assert torch.cuda.memory_allocated() == before


def test_a_written_output_is_noticed():
    """save='input' keeps the output of postnorm_residual: a write to it before
    the backward pass is an error, and without one its gradient is right."""
    x, u = rand(9, 40).requires_grad_(True), rand(9, 40, seed=1).requires_grad_(True)
    out, y = ag.postnorm_residual(x.view(3, 3, 40), u.view(3, 3, 40), norm="none", next_norm="rms", save="input")
    got = torch.autograd.grad(y.square().sum() + out.sum(), [x, u], retain_graph=True)
    v = x + u
    n = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)
    ref = torch.autograd.grad(n.square().sum() + v.sum(), [x, u])
    for a, b in zip(got, ref):  # both in f32
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)
    with torch.no_grad():
        out.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
