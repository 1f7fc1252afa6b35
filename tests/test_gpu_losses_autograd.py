"""The vocabulary loss as a differentiable function."""

from __future__ import annotations

import gc

import pytest
import torch

from tests.test_gpu_losses import BF16, F16, F32, make

pytestmark = pytest.mark.gpu


def ag():
    from rollfast_amd import autograd

    return autograd


def plain(hidden, weight, targets, z_loss, reduction):
    z = torch.matmul(hidden, weight.t())
    lse = torch.logsumexp(z, 1)
    on = targets != -100
    loss = torch.where(on, lse - z.gather(1, torch.where(on, targets, 0)[:, None])[:, 0] + z_loss * lse ** 2, 0.0)
    return loss.sum() if reduction == "sum" else loss.sum() / on.sum()


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("dtype,tol", [(F32, 1e-5), (BF16, 2.0 ** -7), (F16, 2.0 ** -9)])
def test_gradients(dtype, tol, reduction):
    """dz and the gradients are rounded once each, and once more by the loss' own gradient."""
    hidden, weight, targets, _ = make(90, 250, 64, dtype, seed=3, masked=0.2)
    hidden.requires_grad_()
    weight.requires_grad_()
    loss = ag().linear_cross_entropy(hidden, weight, targets, z_loss=1e-3, reduction=reduction)
    (loss * 3.0).backward()
    h, w = hidden.detach().double().cpu().requires_grad_(), weight.detach().double().cpu().requires_grad_()
    ref = plain(h, w, targets.cpu(), 1e-3, reduction)
    (ref * 3.0).backward()
    assert abs(loss.item() - ref.item()) < 1e-5 * abs(ref.item())
    for got, r in ((hidden.grad, h.grad), (weight.grad, w.grad)):
        assert got.dtype == dtype
        assert ((got.double().cpu() - r).norm() / r.norm()).item() < 1.5 * tol


def test_against_differences():
    hidden, weight, targets, _ = make(20, 60, 24, F32, seed=5)
    hidden.requires_grad_()
    weight.requires_grad_()
    ag().linear_cross_entropy(hidden, weight, targets).backward()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    for x in (hidden, weight):
        d = torch.randn(x.shape, generator=gen, device="cuda")
        step = 2.0 ** -7
        with torch.no_grad():
            up, down = (ag().linear_cross_entropy(*((x + s * d if y is x else y) for y in (hidden, weight)), targets)
                        for s in (step, -step))
        # the quotient: f32 losses of about 4 over a step of 2^-6, and a third derivative of order one
        assert abs(((up - down) / (2 * step)).item() - (x.grad * d).sum().item()) < 4 * 2.0 ** -23 / step * 8 + step ** 2 * 10


def test_parts_of_the_gradient_and_none():
    hidden, weight, targets, _ = make(30, 100, 64, BF16, seed=7)
    full = [x.clone().requires_grad_() for x in (hidden, weight)]
    ag().linear_cross_entropy(*full, targets).backward()
    for which in (0, 1):
        args = [hidden, weight]
        args[which] = args[which].clone().requires_grad_()
        ag().linear_cross_entropy(*args, targets).backward()
        assert torch.equal(args[which].grad, full[which].grad)
    loss = ag().linear_cross_entropy(hidden, weight, targets)
    assert not loss.requires_grad
    with torch.no_grad():
        assert torch.equal(ag().linear_cross_entropy(*full, targets), loss)
    out = ag().linear_cross_entropy(*full, targets)
    out.backward(retain_graph=True)  # and again: the kept gradients are as they were
    out.backward()
    assert torch.allclose(full[0].grad.float(), 3 * args[0].float() * 0 + 3 * torch.autograd.grad(
        ag().linear_cross_entropy(*full, targets), full[0])[0].float(), rtol=2.0 ** -6)


def test_autocast_casts_both():
    hidden, weight, targets, _ = make(40, 120, 64, F32, seed=9)
    weight.requires_grad_()
    hidden.requires_grad_()
    with torch.autocast("cuda", dtype=BF16):
        loss = ag().linear_cross_entropy(hidden, weight, targets)
    loss.backward()
    ref = [x.detach().to(BF16).requires_grad_() for x in (hidden, weight)]
    plain_loss = ag().linear_cross_entropy(*ref, targets)
    plain_loss.backward()
    assert torch.equal(loss, plain_loss)
    assert weight.grad.dtype == F32 and torch.equal(weight.grad, ref[1].grad.float())
    assert torch.equal(hidden.grad, ref[0].grad.float())


def test_an_output_dropped_is_freed():
    hidden, weight, targets, _ = make(64, 4000, 256, BF16, seed=11)
    weight.requires_grad_()
    ag().linear_cross_entropy(hidden, weight, targets)
    gc.collect()  # what other tests left
    before = torch.cuda.memory_allocated()
    for _ in range(3):
        ag().linear_cross_entropy(hidden, weight, targets)
    assert torch.cuda.memory_allocated() <= before


def test_a_step_captured_while_an_eager_graph_lives():
    hidden, weight, targets, _ = make(50, 200, 64, F32, seed=13)
    weight.requires_grad_()
    alive = ag().linear_cross_entropy(hidden, weight, targets)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        loss, grad = ag().losses.linear_cross_entropy_grad(hidden, weight.detach(), targets, reduction="mean")[::2]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, alive.detach())
        assert torch.equal(torch.autograd.grad(alive, weight, retain_graph=True)[0], grad)
