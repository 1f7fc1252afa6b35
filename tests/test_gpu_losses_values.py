"""The vocabulary loss where values are far apart: gradients that a loss scale keeps
from being subnormal, tokens that weigh little beside others, confident tokens with
large logits, few tokens that count, infinite logits.  Against the definition in 64
bits; tolerances from the arithmetic, beside each test."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_losses import BF16, F16, F32, HALF_ULP, TINY, U, check, make, near, product, reference, rf

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


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [64, 130, 1000])
def test_confident_tokens_with_large_logits(vocab, dtype):
    """The targets' logits are 50 to 500, all others 200, or 9 to 16, below them, true
    losses zero or 1e-7 to 1e-1.  hidden is the identity and weight holds the logits in a
    few bits, so that they are exact, and the gradient of weight is dz itself.

    exp's argument d is rounded twice (log2(e) is, too): 3 |d| U, and exp2 within 2 ulps;
    s is a sum of a one and at most 1000 terms in f32, its parts rounded in 10 + 16 sums
    of a tile and the blocks': (d 3 + 4 + 26) U of what is added to the one, and U for each
    of the sums that hold the one, 26; log and expm1 within 2 ulps each of their results.
    dz is kept to 22 bits in f32."""
    n = 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(61)
    step = {F32: 2.0 ** -10, F16: 0.25, BF16: 2.0}[dtype]
    top = torch.linspace(50.0, 500.0, n, device="cuda").div(step).round() * step
    # 64 columns: a token each
    far = torch.arange(n, device="cuda") % 2 == 0
    gap = torch.where(far[:, None], 200.0, 9.0 + 7.0 * torch.rand(n, vocab, generator=gen, device="cuda"))
    gap = gap.div(step).round() * step
    z = top[:, None] - gap
    targets = torch.randint(vocab, (n,), generator=gen, device="cuda")
    at = torch.arange(n, device="cuda")
    z[at, targets] = top
    weight = z.t().contiguous().to(dtype)
    assert torch.equal(weight.t().float(), z)
    hidden = torch.eye(n, device="cuda").to(dtype)
    z = z.double()
    p = torch.exp(z - z.amax(1, keepdim=True))
    p[at, targets] = 0.0
    rest = p.sum(1)
    loss = torch.log1p(rest)
    d = (z.amax(1, keepdim=True) - z)
    rel = (3 * d.clamp(max=200) + 30) * U
    bound = 30 * U + (p * rel).sum(1) + 4 * U * loss
    got = rf().linear_cross_entropy_grad(hidden, weight, targets, torch.ones(n, device="cuda"))
    alone = rf().linear_cross_entropy(hidden, weight, targets)
    for x in (got.loss, alone):
        assert (x >= 0).all()
        assert ((x.double() - loss).abs() <= bound).all()
    dz = got.weight.double().t()
    assert (dz[at, targets] <= 0).all()
    half = {F32: 2.0 ** -22 + U, BF16: 2.0 ** -7, F16: 2.0 ** -10}[dtype]  # dz, and the result
    true = -rest / (1 + rest)
    tiny = 2.0 ** -24 if dtype == F16 else 0.0
    assert ((dz[at, targets] - true).abs() <= bound + half * true.abs() + tiny).all()
    if dtype == F32:
        q = p / (1 + rest)[:, None]
        off = q * (rel + 34 * U + half) + 2.0 ** -37  # dz is held down to 2^-38 of a dloss of one
        off[at, targets] = 1.0
        assert ((dz - q).abs() <= off).all()


def spread(tokens, exponents, seed):
    """dloss of either sign, a few powers of two apart."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    e = torch.tensor(exponents, device="cuda")[torch.randint(len(exponents), (tokens,), generator=gen, device="cuda")]
    d = torch.ldexp(1.0 + torch.rand(tokens, generator=gen, device="cuda"), e)
    return torch.where(torch.rand(tokens, generator=gen, device="cuda") < 0.5, d, -d)


def check_rows(hidden, weight, targets, dloss, z_loss=0.0):
    """dhidden row by row against that of a dloss of one, times the row's: as exact as where no
    other token weighs more.  What is held beside a dloss of one is held down to 2^-38 of
    it, or, where another weighs up to 2^5 of it, to 2^-33 (the bound's 2^-38 comes with the reference)."""
    got = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss, z_loss=z_loss)
    loss, (dh, off), dw = reference(hidden, weight, targets, torch.sign(dloss), z_loss)
    near(got.loss, loss, "loss")
    most = (1 + 2 * z_loss * (loss[0].abs().max() + 100)).item()
    off = off + 2.0 ** -33 * most * weight.double().abs().sum(0)
    size = dloss.double().abs()[:, None]
    value, off = dh * size, off * size
    bound = HALF_ULP[got.hidden.dtype] * (value.abs() + off) * 1.01 + TINY[got.hidden.dtype] + off
    assert ((got.hidden.double() - value).abs() <= bound).all()
    return got


@pytest.mark.parametrize("z_loss", [0.0, 1e-2])
@pytest.mark.parametrize("exponents", [(0, -13, -27, -40), (60, 0, -60), (0, -3, -4, -5), (0, -100)])
@pytest.mark.parametrize("size", [(96, 700, 128), (40, 5000, 65), (600, 300, 40)])
def test_f32_tokens_that_weigh_little_keep_their_gradients(size, exponents, z_loss):
    """A power of two for each token.  dweight's sums are right to what the heaviest tokens leave."""
    hidden, weight, targets, _ = make(*size, F32, seed=63, masked=0.1)
    dloss = spread(size[0], exponents, 64)
    got = check_rows(hidden, weight, targets, dloss, z_loss)
    _, _, dw = reference(hidden, weight, targets, dloss, z_loss)
    near(got.weight, dw, "dweight")


def test_f32_dweight_of_tokens_that_weigh_little():
    """A token alone in its column of hidden: dweight's column is its own dz, which is held
    to 22 bits however little it weighs, since hidden's row takes the power of two: ones,
    held as 2^14, of which 2^-20 leaves 2^-6, 19 bits above what is lost, 2^-25."""
    n, vocab = 64, 300
    _, weight, targets, _ = make(n, vocab, n, F32, seed=65)
    hidden = torch.eye(n, device="cuda")
    e = -(torch.arange(n, device="cuda") % 5) * 5
    dloss = torch.ldexp(torch.ones(n, device="cuda"), e)
    got = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    z = weight.double().t()
    dz = torch.softmax(z, 1)
    dz[torch.arange(n, device="cuda"), targets] -= 1
    # of p: the split logits (3 * 2^-22 of at most 64 magnitudes' sum, here one), 16 ulps of exp and sums
    rel = 2.0 ** -22 * 2 + (3 * 2.0 ** -22 + 3 * U) * z.abs().amax(1, keepdim=True) * 4 + (16 + 64 + 6 + 34) * U
    off = dz.abs() * rel + (vocab / 64) * U * dz.abs()
    assert ((got.weight.double().t() / dloss.double()[:, None] - dz).abs() <= off + 2.0 ** -37).all()


@pytest.mark.parametrize("exponents", [(13, -15), (10, 6, 5, 4, -3)])
def test_f16_tokens_that_weigh_little_keep_their_gradients(exponents):
    """weight's rows have a common part, so that what is lost of many small dz shows."""
    hidden, weight, targets, _ = make(300, 5000, 64, F16, seed=67, masked=0.1, logit=0.3)
    weight = (weight.float() + 1.0).to(F16)
    dloss = spread(300, exponents, 68)
    got = check_rows(hidden, weight, targets, dloss)
    _, _, dw = reference(hidden, weight, targets, dloss)
    near(got.weight, dw, "dweight")


def test_tokens_far_apart_in_several_pieces_and_few():
    """Each piece has its own largest; f16's low parts of few tokens are lifted alike."""
    hidden, weight, targets, _ = make(400, 1 << 20, 9, F32, seed=69, masked=0.1)
    dloss = spread(400, (0, -30), 70)
    dloss[:256] *= 2.0 ** -20
    check_rows(hidden, weight, targets, dloss)
    for tokens in (1, 7, 16):
        hidden, weight, targets, _ = make(tokens, 900, 80, F16, seed=71)
        check_rows(hidden, weight, targets, spread(tokens, (8, -4), 72))
        check(hidden, weight, targets, spread(tokens, (8, -4), 72))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_zeros_and_values_that_are_not_finite_in_dloss(dtype):
    """They change no other token's gradient of hidden."""
    hidden, weight, targets, _ = make(50, 200, 64, dtype, seed=73)
    dloss = spread(50, (0, -20) if dtype == F32 else (0, -8), 74)
    ref = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    for value in (0.0, math.nan, math.inf):
        bad = dloss.clone()
        bad[7] = value
        got = rf().linear_cross_entropy_grad(hidden, weight, targets, bad)
        assert not got.hidden[7].any() if value == 0.0 else not got.hidden[7].isfinite().any()
        keep = torch.arange(50, device="cuda") != 7
        assert torch.equal(got.hidden[keep], ref.hidden[keep])


def test_a_graph_replayed_with_other_weights_of_the_tokens():
    hidden, weight, targets, dloss = make(130, 700, 64, F32, seed=75, masked=0.2)
    rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    for turn, exponents in enumerate([(0, -30), (0,), (0, -7), (-90, 0)]):
        dloss.copy_(spread(130, exponents, 80 + turn))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)):
            assert torch.equal(x, y), turn


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens", [20, 129, 500, 3000])
@pytest.mark.parametrize("count", [1, 5, 16])
def test_few_tokens_that_count_among_any_number(count, tokens, dtype):
    """Where at most 16 tokens count their dz keeps twice the bits, however many the call
    has.  dweight's rows that are no target, whose 3900 dz of a token are rounded each on
    its own.  Against r, what rounding the exact gradient costs, the error is 1.01 r for
    bf16, r and an eighth of it from the f16 exponential, and sqrt(2) r for f16, whose
    exponentials are rounded as much; dz rounded to the type would make it sqrt(2) r and
    sqrt(3) r.  The bounds lie halfway."""
    vocab, n = 4000, 96
    hidden, weight, targets, dloss = make(tokens, vocab, n, dtype, seed=91)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(92)
    on = torch.randperm(tokens, generator=gen, device="cuda")[:count]
    off = torch.ones(tokens, dtype=torch.bool, device="cuda")
    off[on] = False
    targets[off] = -100
    dloss = torch.full((tokens,), 1.0, device="cuda")
    got = check(hidden, weight, targets, dloss)
    _, dw = gradients(hidden, weight, targets, dloss)
    rest = torch.ones(vocab, dtype=torch.bool, device="cuda")
    rest[targets[on]] = False
    r = (dw.to(dtype).double() - dw)[rest].norm()
    assert (got.weight.double() - dw)[rest].norm() < {BF16: 1.2, F16: 1.57}[dtype] * r


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_few_tokens_that_count_in_several_pieces(dtype):
    hidden, weight, targets, dloss = make(2100, 1 << 20, 16, dtype, seed=93)
    keep = targets[[3, 1900]].clone()
    targets[:] = -100
    targets[[3, 1900]] = keep
    got = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    rows = torch.tensor([3, 1900], device="cuda")
    alone = rf().linear_cross_entropy_grad(hidden[rows].contiguous(), weight, targets[rows].contiguous(), dloss[rows].contiguous())
    assert torch.equal(got.loss[rows], alone.loss) and torch.equal(got.hidden[rows], alone.hidden)
    assert not got.hidden[targets == -100].any()
    assert ((got.weight.double() - alone.weight.double()).norm() <= 2 * HALF_ULP[dtype] * alone.weight.double().norm()).item()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens", [6, 40, 300])
def test_infinite_logits_of_16_bit_tensors(tokens, dtype):
    """An entry of -inf is not there: losses and the other rows' gradients are those of
    the table without it (sums may be in another order: twice the bounds), its own
    gradient zero.  One of +inf makes its token's loss and gradients not finite, and no
    other token's."""
    hidden, weight, targets, dloss = make(tokens, 90, 8, dtype, seed=19)
    hidden[:, 0] = hidden[:, 0].abs() + 0.125
    weight[11] = 0.0
    weight[11, 0] = -math.inf
    targets[targets == 11] = 3
    keep = torch.arange(90, device="cuda") != 11
    less = weight[keep].contiguous()
    moved = torch.where(targets > 11, targets - 1, targets)
    loss, _, dw = reference(hidden, less, moved, dloss)
    got = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    for x in (got.loss, rf().linear_cross_entropy(hidden, weight, targets)):
        near(x, (loss[0], 2 * loss[1]), "loss")
    near(got.weight[keep], (dw[0], 2 * dw[1]), "dweight")
    assert not got.weight[11].any()
    hidden[2, 0] = -1.0  # its logit 11 is +inf
    bad = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    other = torch.arange(tokens, device="cuda") != 2
    assert torch.equal(bad.loss[other], got.loss[other])
    assert not bad.loss[2].isfinite() and not bad.hidden[2].isfinite().any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_a_row_of_hidden_that_is_not_finite(dtype):
    """A row of hidden with a NaN or an Inf: its loss is not finite, the others' as they were."""
    hidden, weight, targets, dloss = make(20, 150, 16, dtype, seed=21)
    ref = rf().linear_cross_entropy(hidden, weight, targets)
    for value in (math.nan, math.inf):
        bad = hidden.clone()
        bad[5, 3] = value
        got = rf().linear_cross_entropy_grad(bad, weight, targets, dloss)
        other = torch.arange(20, device="cuda") != 5
        assert torch.equal(got.loss[other], ref[other]) or dtype == F32
        assert got.loss[other].isfinite().all() and got.hidden[other].isfinite().all()
        assert not got.loss[5].isfinite() and not got.weight.isfinite().all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_forward_and_backward_in_one_graph(dtype):
    """Captured together, replayed with other inputs and other work between, against eager
    calls on leaves of their own."""
    from rollfast_amd import autograd

    def step(h, w, t, scale):
        loss = autograd.linear_cross_entropy(h, w, t, z_loss=1e-3)
        return (loss.detach(), *torch.autograd.grad(loss * scale, (h, w)))

    hidden, weight, targets, _ = make(130, 700, 64, dtype, seed=95, masked=0.2)
    scale = torch.full((), 2.0 ** 10, device="cuda")
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(h, w, targets, scale)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(h, w, targets, scale)
    for turn in range(4):
        h2, w2, t2, _ = make(130, 700, 64, dtype, seed=300 + turn, masked=0.1 * turn)
        with torch.no_grad():
            h.copy_(h2)
            w.copy_(w2)
            targets.copy_(t2)
            scale.fill_(2.0 ** (10 + turn))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, step(h2.requires_grad_(), w2.requires_grad_(), t2, scale)):
            assert torch.equal(x, y), turn


def test_f16_tokens_far_apart_in_several_pieces():
    """Pieces of 768 tokens: dhidden as from calls on their tokens alone, dweight their sum."""
    hidden, weight, targets, _ = make(1100, 1 << 20, 8, F16, seed=97, masked=0.1)
    dloss = spread(1100, (9, -9), 98)
    got = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    total = torch.zeros(weight.shape, dtype=torch.float64, device="cuda")
    for part in (slice(0, 400), slice(400, 1100)):
        one = rf().linear_cross_entropy_grad(hidden[part], weight, targets[part], dloss[part])
        total += one.weight.double()
        # four roundings of 2^-10 / sqrt(12) on either side, in rows of eight
        assert rows_off(got.hidden[part], one.hidden.double()) < 2.0 ** -9
    # of A, the sum of the terms' magnitudes: dz is rounded, 2^-11, on either side (at scales
    # that differ), the parts and the whole are, and sums of up to 1100 terms; f16's own
    # steps below 2^-14 are 2^-24, three times halved
    rows = torch.nonzero(targets != -100)[:, 0]
    h, d = hidden[rows].double().abs(), dloss[rows].double().abs()
    z = torch.softmax(product(hidden[rows].double(), weight.double()), 1)
    z[torch.arange(len(rows), device="cuda"), targets[rows]] += 1
    a = torch.matmul((z * d[:, None]).t().contiguous(), h)
    assert ((got.weight.double() - total).abs() <= (4 * 2.0 ** -11 + 2 * 1180 * U) * a + 2.0 ** -23).all()
