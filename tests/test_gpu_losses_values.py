"""The vocabulary loss where values are far apart: gradients that a loss scale keeps
from being subnormal, tokens that weigh little beside others, confident tokens with
large logits, few tokens that count, infinite logits.  Against the definition in 64
bits; tolerances from the arithmetic, beside each test."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_losses import BF16, F32, make, rf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [1.0 / 3.0, 2.0 ** 17, 1e-3])
def test_the_loss_gradient_is_not_rounded_first(scale, dtype):
    """What the backward pass multiplies by is f32, whatever the gradients are."""
    from rollfast_amd import autograd

    hidden, weight, targets, _ = make(50, 120, 40, dtype, seed=57, masked=0.2)
    kept = rf().linear_cross_entropy_grad(hidden, weight, targets, reduction="sum")
    h, w = (x.clone().requires_grad_() for x in (hidden, weight))
    (autograd.linear_cross_entropy(h, w, targets, reduction="sum") * scale).backward()
    for got, one in ((h.grad, kept.hidden), (w.grad, kept.weight)):
        assert torch.equal(got, (one.float() * torch.tensor(scale, device="cuda")).to(dtype))
