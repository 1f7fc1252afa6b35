"""The orthogonalisation of matrices against its definition in 64 bits.

What a rounding in a step does to the result depends on the matrix, so the bounds
are of the 2-norm of the difference over that of the result, and stated for
matrices whose result has a norm of the order of sqrt(n): the steps' map has a
derivative of at most a = 3.4445 at each step, 485 over five, and only towards
singular values that are still small, whose part of the norm is as small.
- bfloat16 results: the last rounding is off by at most half an ulp, 2^-8 of every
  value and so of the norm (in small matrices it does not average out: a column of
  five values has been off by 3.1e-3).  The products' roundings to float16, 2^-11 at
  most each, reach the result through (b A + c A^2) X with a factor of at most
  |B| = 4.8 in one of 5 steps and 2.8 in the others, and average out over n terms:
  2 * 2^-11 * (4.8 + 4 * 2.8) / sqrt(3) / 4 = 2.3e-3 together.  2^-8 + 2.3e-3 = 6.2e-3.
- float32 results: split numbers of 22 bits and sums of f32 in every product: an
  error of 2^-22 + sqrt(k) U of each entry, times 485 at worst for what is small
  and about 10 for what is not: 2e-5 covers k up to 4096.
- float16: that and the rounding, 2^-11: 5.1e-4.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
BOUND = {BF16: 6.2e-3, F32: 2e-5, F16: 5.1e-4}


def rf():
    import rollfast_amd

    return rollfast_amd


def gaussian(rows, cols, dtype, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return (torch.randn(rows, cols, generator=gen, device="cuda") * scale).to(dtype)


def low_rank(rows, cols, dtype, seed=0, noise=0.02):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    k = max(1, min(rows, cols, 64) // 2)
    left = torch.randn(rows, k, generator=gen, device="cuda") * torch.exp(-torch.arange(k, device="cuda") / 8.0)
    x = left @ torch.randn(k, cols, generator=gen, device="cuda")
    return (x + noise * torch.randn(rows, cols, generator=gen, device="cuda")).to(dtype)


def exact(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = (x.t() if tall else x).contiguous()
    x = x / (x.norm() + eps)
    table = coefficients if isinstance(coefficients[0], tuple) else [coefficients] * steps
    for a, b, c in table:
        k = torch.matmul(x, x.t().contiguous())
        x = a * x + torch.matmul(b * k + c * torch.matmul(k, k), x)
    return x.t() if tall else x


def off(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


SIZES = [(1, 1), (1, 7), (5, 1), (3, 5), (31, 64), (64, 64), (65, 63), (100, 700), (300, 129), (256, 768), (517, 301),
         (128, 2049), (1025, 260), (640, 640)]


@pytest.mark.parametrize("dtype", [BF16, F32, F16])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("kind", [gaussian, low_rank])
def test_sizes(kind, size, dtype):
    g = kind(*size, dtype, seed=size[0])
    got = rf().orthogonalize(g)
    assert got.dtype == dtype and got.shape == g.shape
    assert off(got, exact(g)) < BOUND[dtype]


def test_a_list_in_one_call():
    for dtype in (BF16, F32):
        tree = {"a": [gaussian(r, c, dtype, seed=i) for i, (r, c) in enumerate(SIZES * 3)], "b": (low_rank(90, 40, F16),)}
        got = rf().orthogonalize(tree)
        for g, x in zip(tree["a"], got["a"]):
            assert off(x, exact(g)) < BOUND[dtype]
        assert off(got["b"][0], exact(tree["b"][0])) < BOUND[F16]


def test_steps_coefficients_and_scale():
    g = gaussian(96, 200, F32)
    for steps in (0, 1, 2, 7):
        assert off(rf().orthogonalize(g, steps=steps), exact(g, steps)) < BOUND[F32]
    rows = ((3.0, -3.2, 1.2), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375))
    assert off(rf().orthogonalize(g, steps=3, coefficients=rows), exact(g, 3, rows)) < BOUND[F32]
    assert off(rf().orthogonalize(g, scale=-2.5), -2.5 * exact(g)) < BOUND[F32]
    assert off(rf().orthogonalize(g, eps=100.0), exact(g, eps=100.0)) < BOUND[F32]
