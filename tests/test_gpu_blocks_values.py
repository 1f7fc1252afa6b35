"""Residual-block operators at values where an overflow, a lost digit or an
infinity of one operand must not reach a result that does not depend on it.
U is half an f32 ulp, 2^-24."""

from __future__ import annotations

import math

import pytest
import torch

import rollfast_amd as rf

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rand(*shape, dtype=F32, seed=0, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_activation_slopes_of_large_values(name, dtype):
    """Up to the type's largest value act(x) is x or 0 and its slope 1 or 0."""
    top = torch.finfo(dtype).max
    v = [s for s in (1e3, 1e4, 6e4, 1e9, 1.9e19, 1e25, 1e30, 1e38) if s < top] + [top]
    x = torch.tensor([v + [-s for s in v]], dtype=dtype, device="cuda")
    up, dh = torch.full_like(x, 0.5), torch.full_like(x, 2.0)
    on = (x > 0).to(dtype)
    h, saved = rf.gated_activation(x, up, activation=name, save="input")
    assert torch.equal(h, on * x * up)
    dg, du = rf.gated_activation_grad(dh, saved)
    assert torch.equal(dg, on), dg
    assert torch.equal(du, torch.where(x > 0, dh * x, torch.zeros_like(x))), du
