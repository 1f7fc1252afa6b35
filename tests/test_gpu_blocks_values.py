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


def test_silu_keeps_f32s_digits():
    """f32's SiLU and its slope in relative terms, on the negative tail too.
    exp is within an ulp (2 U), 1 + e and the quotient within U each, the two
    products within U each, which is 6 U for h and for dup; the slope adds the
    difference, the fused product and, by its condition |x| / (|x| - 1) <= 4 / 3
    for x <= -4, a third of what came before: below 12 U.  16 U for all.  On the
    positive side the slope's s is off by 1.5 U of 1 and 1 - s by as much, which
    x (1 - s) multiplies by x, up to the x of about 17 where s is 1: 2 U x more."""
    x = torch.cat((torch.linspace(-80, -4, 4001), torch.linspace(4, 80, 4001))).cuda()[None]
    up, dh = rand(1, 8002, seed=1) + 3.0, rand(1, 8002, seed=2) - 4.0
    h, saved = rf.gated_activation(x, up, save="input")
    dg, du = rf.gated_activation_grad(dh, saved)
    x64, u64, d64 = x.double(), up.double(), dh.double()
    s = 1 / (1 + torch.exp(-x64))
    for got, ref, what in ((h, x64 * s * u64, "h"), (du, d64 * x64 * s, "dup"),
                           (dg, d64 * u64 * s * (1 + x64 * (1 - s)), "dgate")):
        off = ((got.double() - ref) / ref).abs()
        bound = 16 * U + (2 * U * x64.clamp(0, 18) if what == "dgate" else 0)
        assert (off <= bound).all(), (what, (off.max() / U).item(), x.flatten()[off.argmax()].item())


@pytest.mark.parametrize("shape", [(3, 5), (9, 40), (5, 301), (4, 1283), (6, 4096), (3, 5000), (4, 9000), (3, 16411)])
@pytest.mark.parametrize("gate", [None, "one", "rows"])
@pytest.mark.parametrize("save", ["int8", "input"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_branch_that_is_not_finite_without_a_norm(shape, gate, save, dtype):
    """norm='none': the gradients at the branch and the residual do not depend
    on the branch's values, so an Inf or NaN in it changes neither; the gate's
    does, in the columns of its checkpoint's block at most."""
    rows, cols = shape
    r, u, dout = (rand(rows, cols, dtype=dtype, seed=i) for i in range(3))
    g = None if gate is None else rand(cols, seed=3) if gate == "one" else rand(rows, cols, seed=3)
    u[0, 1], u[1, cols - 1], u[2, cols // 2] = math.inf, -math.inf, math.nan
    out, _, saved = rf.postnorm_residual(r, u, gate=g, norm="none", branch_scale=0.5, residual_scale=2.0, save=save)
    got = rf.postnorm_residual_grad(dout, None, saved)
    assert torch.equal(got.residual, 2 * dout)
    ref = 0.5 * dout.double() * (1.0 if g is None else g.double())
    half = U if dtype == F32 else 2.0 ** -8
    off = (got.branch.double() - ref).abs()
    assert (off <= 1.01 * (half + U) * ref.abs()).all()  # one product in f32, rounded once
    if g is not None:
        block = torch.arange(cols) // 32
        hit = (block == 0) | (block == (cols - 1) // 32) | (block == cols // 2 // 32)
        assert torch.isfinite(got.gate[..., ~hit]).all()
