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


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_under_autocast(dtype, bias):
    """f32 tensors under autocast: the product has autocast's dtype, x's and
    the bias's gradients are those of torch's linear (within 2^-7 of the norm:
    a rounding of the factors and of the sum to eight bits each, and the
    orders of summation), the weight's is an f32 sum over the checkpoint
    (within 3 % of the norm: steps of 1 / 64 .. 1 / 128 of a block's largest
    value)."""
    x0, w0, b0, dy = rand(70, 96), rand(160, 96, seed=1), rand(160, seed=2), rand(70, 160, seed=3)
    got = []
    for f in (ag.linear, torch.nn.functional.linear):
        x, w, b = (t.clone().requires_grad_(True) for t in (x0, w0, b0))
        with torch.autocast("cuda", dtype=dtype):
            y = f(x, w, b if bias else None)
        assert y.dtype == dtype
        y.backward(dy.to(dtype))
        got.append((y.float(), x.grad, w.grad, *((b.grad,) if bias else ())))
        assert all(t.dtype == F32 for t in got[-1])
    for a, b, bound in zip(*got, (2.0 ** -7, 2.0 ** -7, 0.03, 2.0 ** -7)):
        assert (a - b).norm() <= bound * b.norm()


def test_linear_leaves_nothing_in_the_autocast_cache():
    """A weight that autograd.linear and torch's linear share gets the gradient
    of both, whichever comes first under autocast."""
    x, w, dy = rand(40, 64), rand(32, 64, seed=1).requires_grad_(True), rand(40, 32, seed=2, dtype=BF16)
    grads = []
    for order in ((ag.linear, torch.nn.functional.linear), (torch.nn.functional.linear, ag.linear)):
        w.grad = None
        with torch.autocast("cuda", dtype=BF16):
            y = [f(x, w) for f in order]
        torch.autograd.backward(y, [dy, dy])
        grads.append(w.grad.clone())
    ref = 2 * dy.double().t().contiguous().matmul(x.double())
    for g in grads:  # half of it from 8 bits, half rounded to bf16
        assert (g.double() - ref).norm() <= 0.03 * ref.norm()


def test_a_block_under_autocast_trains():
    """The block of the module's docstring in f32 under autocast: every
    parameter has an f32 gradient within 5 % of the norm of the one in f32
    (3 % from 8 bits as without autocast, the rest the bf16 products)."""
    cols, ffn = 96, 160
    p = {"w": 1 + rand(cols, scale=0.1), "gu": rand(2 * ffn, cols, seed=2, scale=0.1),
         "dn": rand(cols, ffn, seed=3, scale=0.1), "w2": 1 + rand(cols, seed=6, scale=0.1)}
    x = rand(5, 14, cols, seed=7)
    co, cy = rand(*x.shape, seed=8), rand(*x.shape, seed=9)
    for v in (*p.values(), x):
        v.requires_grad_(True)

    def block():
        y, k = ag.prenorm(x, p["w"], checkpoint_output=True)
        h, k = ag.gated_activation(ag.linear(y, p["gu"], checkpoint=k), checkpoint_output=True)
        return ag.postnorm_residual(x, ag.linear(h, p["dn"], checkpoint=k), norm="none", next_norm="rms",
                                    next_weight=p["w2"])

    def grads():
        out, y = block()
        return torch.autograd.grad((out * co).sum() + (y.float() * cy).sum(), [x, *p.values()])

    ref = grads()
    with torch.autocast("cuda", dtype=BF16):
        got = grads()
    for name, a, b in zip(["x", *p], got, ref):
        assert a.dtype == F32 and (a - b).norm() <= 0.05 * b.norm(), (name, ((a - b).norm() / b.norm()).item())


class NoGradient(torch.autograd.Function):
    """Passes its input on, and no gradient back."""

    @staticmethod
    def forward(ctx, x):
        return x * 1

    @staticmethod
    def backward(ctx, g):
        return None


def test_outputs_without_a_gradient():
    """No gradient comes back through an output: none goes on."""
    x, w = rand(9, 40).requires_grad_(True), rand(40, seed=1).requires_grad_(True)
    for f in (lambda t: ag.prenorm(t, w), lambda t: ag.gated_activation(t, t),
              lambda t: ag.postnorm_residual(t, t, w),
              lambda t: sum(ag.postnorm_residual(t, t, w, next_norm="rms")), lambda t: ag.linear(t, w[None] * 1)):
        x.grad = w.grad = None
        (NoGradient.apply(f(x)).sum() + x.sum()).backward()
        assert torch.equal(x.grad, torch.ones_like(x)) and (w.grad is None or not w.grad.any())


def test_main_gradient_written_is_noticed():
    """linear_weight_grad writes `out` in place, and says so to autograd."""
    x, dy = rand(20, 64, dtype=BF16), rand(20, 32, dtype=BF16, seed=1)
    kept = blocks.checkpoint_activations(x)
    main = torch.zeros(32, 64, device="cuda")
    a = rand(32, 64, seed=2).requires_grad_(True)
    for accumulate in (False, True):
        y = (a * main).sum()
        version = main._version
        assert blocks.linear_weight_grad(dy, kept, out=main, accumulate=accumulate) is main
        assert main._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        other = torch.zeros(32, 64, device="cuda")
    blocks.linear_weight_grad(dy, kept, out=other)
    assert torch.equal(other, blocks.linear_weight_grad(dy, kept, dtype=F32))
