"""The differentiable forms of the residual-block operators where they need no
GPU: the linear layer with a frozen weight, and refusals."""

from __future__ import annotations

import pytest
import torch

from rollfast_amd import autograd as ag
from rollfast_amd import blocks


def rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_under_autocast(dtype):
    """The product is autocast's, and so is the gradient at x: the same two
    roundings to 16 bits, so the same bits as torch's linear."""
    w, b = rand(3, 7, seed=1), rand(3, seed=2)
    grads = []
    for f in (ag.linear, torch.nn.functional.linear):
        x = rand(5, 7).requires_grad_(True)
        with torch.autocast("cpu", dtype=dtype):
            y = f(x, w, b)
        assert y.dtype == dtype
        y.backward(rand(5, 3, seed=3).to(dtype))
        grads.append((y, x.grad))
    assert grads[0][1].dtype == torch.float32
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


def test_linear_keeps_nothing_where_no_gradient_is_wanted(monkeypatch):
    def made(x):
        raise AssertionError("a checkpoint was made")

    monkeypatch.setattr(blocks, "checkpoint_activations", made)
    x, w, b = rand(5, 7), torch.nn.Parameter(rand(3, 7, seed=1)), torch.nn.Parameter(rand(3, seed=2))
    with torch.no_grad():
        assert torch.equal(ag.linear(x, w, b), torch.nn.functional.linear(x, w, b))
    assert torch.equal(ag.linear(x, w.detach()), torch.nn.functional.linear(x, w.detach()))


def test_gradients_need_something_kept():
    x = rand(4, 8).requires_grad_(True)
    for call in (lambda: ag.prenorm(x, save=None), lambda: ag.postnorm_residual(x, x, save=None),
                 lambda: ag.gated_activation(x, x, save=None)):
        with pytest.raises(ValueError, match="save must be 'int8' or 'input'"):
            call()
