"""The vocabulary loss where values are far apart: gradients that a loss scale keeps
from being subnormal, tokens that weigh little beside others, confident tokens with
large logits, few tokens that count, infinite logits.  Against the definition in 64
bits; tolerances from the arithmetic, beside each test."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_losses import BF16, F16, F32, make, product, rf

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


def gradients(hidden, weight, targets, dloss, z_loss=0.0):
    """(dhidden, dweight) in 64 bits."""
    rows = torch.nonzero(targets != -100)[:, 0]
    h, w = hidden[rows].double(), weight.double()
    z = product(h, w)
    lse = torch.logsumexp(z, 1, keepdim=True)
    dz = torch.exp(z - lse) * (1 + 2 * z_loss * lse)
    dz[torch.arange(len(rows), device="cuda"), targets[rows]] -= 1
    dz *= dloss[rows].double()[:, None]
    dh = torch.zeros(hidden.shape, dtype=torch.float64, device="cuda")
    dh[rows] = torch.matmul(dz, w)
    return dh, torch.matmul(dz.t().contiguous(), h)


def rows_off(got, ref):
    """The largest error of a row, as a part of its norm."""
    norm = ref.norm(dim=1)
    return ((got.double() - ref).norm(dim=1)[norm > 0] / norm[norm > 0]).max().item()


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("cast", [False, True])
def test_a_loss_scale_reaches_f16_gradients(cast, reduction):
    """A mean over 4096 tokens: the gradients are some 1e-6, dweight's of rows that are
    no target 1e-7 and less, where f16 has steps of 6e-8.  A scale of 2^16 (a sum: 2^4)
    brings them back before they are rounded.  Three roundings to f16 (the exponential,
    the logit's gradient, the result), each off by 2^-10 / sqrt(12) = 2.8e-4 of its value
    in the mean, the first two of independent terms: 4.9e-4 together, and twice that is
    allowed for the worst of 20011 rows."""
    hidden, weight, targets, _ = make(4096, 20011, 256, F16, seed=51, masked=0.1, logit=0.3)
    scale = 2.0 ** 16 if reduction == "mean" else 2.0 ** 4
    count = int((targets != -100).sum()) if reduction == "mean" else 1
    dh, dw = gradients(hidden, weight, targets, torch.full((4096,), scale / count, device="cuda"))
    h, w = ((x.float() if cast else x).requires_grad_() for x in (hidden, weight))
    with torch.autocast("cuda", dtype=F16, enabled=cast):
        from rollfast_amd import autograd

        loss = autograd.linear_cross_entropy(h, w, targets, reduction=reduction)
    (loss * scale).backward()
    assert h.grad.dtype == w.grad.dtype == (F32 if cast else F16)
    assert not h.grad[targets == -100].any()
    assert rows_off(h.grad, dh) < 1e-3
    assert rows_off(w.grad, dw) < 1e-3


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,vocab,n", [(70, 300, 72), (1, 1000, 33), (300, 9001, 128), (0, 50, 8)])
def test_f32_gradients_of_16_bit_tensors(tokens, vocab, n, dtype):
    """What the differentiable loss keeps of f16 tensors: the same sums, not rounded."""
    from rollfast_amd import losses

    hidden, weight, targets, _ = make(tokens, vocab, n, dtype, seed=53, masked=0.3)
    wide = losses._call(hidden, weight, targets, None, -100, 1e-3, "sum", True, wide=True)
    ref = rf().linear_cross_entropy_grad(hidden, weight, targets, z_loss=1e-3, reduction="sum")
    assert torch.equal(wide[0], ref.loss)
    for x, y in zip(wide[1:], ref[1:]):
        assert x.dtype == F32 and torch.equal(x.to(dtype), y)
    # the same through the Python host path, from tensors that it lays out
    again = losses._call(hidden.t().contiguous().t(), weight, targets, None, -100, 1e-3, "sum", True, wide=True)
    for x, y in zip(wide, again):
        assert torch.equal(x, y)


def test_f32_gradients_of_several_pieces():
    """The pieces' sums are added in the output itself."""
    from rollfast_amd import losses

    hidden, weight, targets, _ = make(1100, 1 << 20, 16, F16, seed=55, masked=0.1)
    wide = losses._call(hidden, weight, targets, None, -100, 0.0, "mean", True, wide=True)
    ref = rf().linear_cross_entropy_grad(hidden, weight, targets, reduction="mean")
    for x, y in zip(wide[1:], ref[1:]):
        assert x.dtype == F32 and torch.equal(x.to(F16), y)
