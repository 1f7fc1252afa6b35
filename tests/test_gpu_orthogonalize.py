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
  (The result is rounded to float16 before it is rounded to bfloat16, up to 2^-11
  more: not added, the bound stays.)
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


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(dtype):
    g = gaussian(70, 130, dtype, seed=3)
    ref = rf().orthogonalize(g)
    wide = torch.full((70, 150), math.nan, dtype=dtype, device="cuda")
    wide[:, 7:137] = g
    assert torch.equal(rf().orthogonalize(wide[:, 7:137]), ref)
    assert torch.equal(rf().orthogonalize(g.t().contiguous().t()), ref)
    assert torch.equal(rf().orthogonalize(torch.nn.Parameter(g)), ref)
    buffer = torch.empty(70 * 130 + 1, dtype=dtype, device="cuda")
    buffer[1:] = g.reshape(-1)
    assert torch.equal(rf().orthogonalize(buffer[1:].view(70, 130)), ref)
    # the transposed matrix: the same products, read and written the other way round
    assert torch.equal(rf().orthogonalize(g.t()), ref.t())
    # stacked matrices
    other = gaussian(70, 130, dtype, seed=4)
    both = rf().orthogonalize(torch.stack((g, other)).view(1, 2, 70, 130))
    assert both.shape == (1, 2, 70, 130) and torch.equal(both[0, 0], ref)
    assert off(both[0, 1], exact(other)) < BOUND[dtype]
    one = rf().orthogonalize(g[:1].expand(70, 130))
    assert off(one, exact(g[:1].expand(70, 130))) < BOUND[dtype]


def test_nothing_and_zeros():
    assert rf().orthogonalize([]) == []
    for shape in ((0, 5), (5, 0), (0, 3, 4)):
        assert rf().orthogonalize(torch.empty(shape, device="cuda")).shape == shape
    zero = torch.zeros(30, 50, device="cuda")
    assert not rf().orthogonalize(zero).any()
    assert not rf().orthogonalize(zero.to(BF16)).any()
    assert rf().orthogonalize(zero, eps=0.0).isnan().all()


@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_stays_in_its_matrix(junk):
    a, b, c = (gaussian(90, 200, BF16, seed=i) for i in range(3))
    bad = b.clone()
    bad[3, 4] = junk
    x, y, z = rf().orthogonalize([a, bad, c])
    assert torch.equal(x, rf().orthogonalize([a, b, c])[0]) and torch.equal(z, rf().orthogonalize([a, b, c])[2])
    assert y.isnan().all()


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e25])
def test_small_and_large_values(scale):
    g = gaussian(65, 100, F32, seed=5) * scale
    assert off(rf().orthogonalize(g, eps=0.0), exact(g, eps=0.0)) < BOUND[F32]


def test_near_rank_one():
    """What float16 rounds away from X must not be lost: it grows 485 times."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(6)
    for noise in (1e-2, 1e-3, 1e-4):
        g = torch.randn(512, 1, generator=gen, device="cuda") @ torch.randn(1, 700, generator=gen, device="cuda")
        g = (g + noise * torch.randn(512, 700, generator=gen, device="cuda")).to(BF16)
        assert off(rf().orthogonalize(g), exact(g)) < BOUND[BF16]


def test_long_thin_and_many():
    for shape in ((3, 100000), (200000, 2)):
        g = gaussian(*shape, BF16, seed=8)
        assert off(rf().orthogonalize(g), exact(g)) < BOUND[BF16]
    many = [gaussian(1 + i % 70, 3 + i % 45, (BF16, F32, F16)[i % 3], seed=i) for i in range(301)]
    for g, x in zip(many, rf().orthogonalize(many)):
        assert off(x, exact(g)) < BOUND[g.dtype]


def test_tiles_of_256_and_split_sums():
    """Large enough for whole rounds, a last round in parts, and both kinds of tiles."""
    for dtype in (BF16, F32):
        matrices = [gaussian(1100, 3000, dtype, seed=1), gaussian(2100, 2100, dtype, seed=2), gaussian(3001, 700, dtype, seed=3)]
        for g, x in zip(matrices, rf().orthogonalize(matrices)):
            assert off(x, exact(g)) < BOUND[dtype]
        for g in matrices:
            assert off(rf().orthogonalize(g), exact(g)) < BOUND[dtype]


def test_equal_inputs_give_equal_bits():
    g = [gaussian(700, 900, BF16, seed=1), gaussian(300, 200, BF16, seed=2)]
    first = rf().orthogonalize(g)
    for _ in range(3):
        for x, y in zip(rf().orthogonalize(g), first):
            assert torch.equal(x, y)


def test_another_stream_and_a_graph():
    g = gaussian(200, 333, BF16, seed=1)
    ref = rf().orthogonalize(g)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = rf().orthogonalize(g)
    stream.synchronize()
    assert torch.equal(got, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rf().orthogonalize(g)
    for turn in range(4):
        other = gaussian(200, 333, BF16, seed=50 + turn)
        g.copy_(other)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, rf().orthogonalize(other)), turn


@pytest.mark.parametrize("dtype", [BF16, F32, F16])
def test_rows_that_share_memory(dtype):
    g = gaussian(1, 96, dtype)
    wide = g.expand(40, 96)
    # rank one: its only singular value is the norm
    assert off(rf().orthogonalize(wide), exact(wide.contiguous())) < BOUND[dtype]
    table = gaussian(300, 64, dtype, seed=1)
    rows = table.as_strided((120, 64), (16, 1))
    assert off(rf().orthogonalize(rows), exact(rows.contiguous())) < BOUND[dtype]
    got = rf().orthogonalize([table, table])
    assert torch.equal(got[0], got[1]) and got[0].data_ptr() != got[1].data_ptr()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_matrix_of_each_tile(dtype):
    """From sides that tiles of 64 share out to ones that fill the GPU with tiles of 256."""
    for r, c in ((200, 330), (390, 1300), (1000, 1100), (1700, 2600)):
        g = low_rank(r, c, dtype, seed=r, noise=0.2)
        assert off(rf().orthogonalize(g), exact(g)) < BOUND[dtype], (r, c)


def test_stacks_without_elements():
    """An empty stack, stacked matrices without rows or without columns, among others."""
    g = gaussian(20, 30, F32)
    shapes = [(0, 3, 4), (2, 0, 4), (2, 3, 0), (2, 0, 0, 5), (0, 4), (3, 0)]
    got = rf().orthogonalize([torch.empty(s, device="cuda") for s in shapes] + [g])
    assert [tuple(x.shape) for x in got[:-1]] == shapes and torch.equal(got[-1], rf().orthogonalize(g))
