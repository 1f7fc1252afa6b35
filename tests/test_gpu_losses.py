"""The vocabulary loss against its definition in 64 bits.

Tolerances are bounds on the arithmetic, stated before any run.  U is half an f32
ulp, 2^-24; n the hidden size.
- A logit is a sum of n exact products in f32: off by at most (n + 8) U of the sum of
  their magnitudes.  f32 tensors are split into two f16 parts: each is off by 2^-22
  of its value, and low times low (2^-22 of the product) is left out: 3 * 2^-22 more;
  below 2^-25 of a scaled value, 2^-39 of the tensor's largest, a part is lost.
- exp is within FEW ulps and 2 |x| U for the product with log2(e); the sums of 128
  exponentials, of a lane's blocks and of a wave: (128 + blocks + 64) U.
- An exponential kept in f16 is off by 2^-11 of its value and 2^-25; dz is rounded
  once to the tensors' type (f32: to 2^-22), below 2^-25 of a value scaled to 2^14
  for f16 and f32.
- The products with dz are sums of vocab or tokens terms in f32, in up to 64 parts,
  and several pieces; the gradient is rounded once to its type.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FEW = 16
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_ULP = {F32: U, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}
KEPT = {F32: 2.0 ** -22, BF16: 2.0 ** -8, F16: 2.0 ** -11}  # dz before its products


def rf():
    import rollfast_amd

    return rollfast_amd


def make(tokens, vocab, n, dtype, seed=0, masked=0.0, logit=1.0, ignore=-100, kind=torch.int64):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    hidden = torch.randn(tokens, n, generator=gen, device="cuda")
    weight = torch.randn(vocab, n, generator=gen, device="cuda") * (logit / math.sqrt(n))
    targets = torch.randint(vocab, (tokens,), generator=gen, device="cuda")
    targets[torch.rand(tokens, generator=gen, device="cuda") < masked] = ignore
    dloss = torch.randn(tokens, generator=gen, device="cuda") / max(1, tokens)
    return hidden.to(dtype), weight.to(dtype), targets.to(kind), dloss


def product(a, b):
    """a b^T in 64 bits."""
    return torch.matmul(a, b.t().contiguous())


def reference(hidden, weight, targets, dloss, z_loss=0.0, ignore=-100):
    """(loss, dhidden, dweight) in 64 bits and bounds on their errors before the last rounding."""
    dtype, n, vocab = hidden.dtype, hidden.shape[1], weight.shape[0]
    h, w = hidden.double(), weight.double()
    on = targets != ignore
    rows = torch.nonzero(on)[:, 0]
    h, y, dl = h[rows], targets[rows].long(), dloss[rows].double()
    z, size = product(h, w), product(h.abs(), w.abs())
    off = (n + 8) * U * size
    if dtype == F32:
        off = off * 3 + 3 * 2.0 ** -22 * size  # three sums
        top = 2.0 ** -39 * (h.abs().max() * w.abs().sum(1).max() + w.abs().max() * h.abs().sum(1).max()) if len(rows) else 0.0
        off = off + top
    lse = torch.logsumexp(z, 1)
    at = torch.arange(len(rows), device=z.device)
    zt = z[at, y]
    far = off.amax(1) if len(rows) else off.sum(1)
    spread = (z.amax(1, keepdim=True) - z) if len(rows) else z
    blocks = vocab / 64 + 1
    summed = (128 + blocks + 64 + FEW) * U + ((spread * 4 * U) * torch.exp(z - lse[:, None])).sum(1)
    one = 2 * far + summed + 8 * U * (lse.abs() + zt.abs() + z.abs().amax(1) if len(rows) else lse)
    loss = torch.zeros(len(targets), dtype=torch.float64, device=z.device)
    loss_off = loss.clone()
    loss[rows] = lse - zt + z_loss * lse ** 2
    loss_off[rows] = one * (1 + 2 * z_loss * lse.abs()) + 4 * U * z_loss * lse ** 2
    p = torch.exp(z - lse[:, None])
    grow = 1 + 2 * z_loss * lse[:, None]
    dz = p * grow
    dz[at, y] -= 1
    dz = dz * dl[:, None]
    # of p: the errors of its logit and of lse, an f16 rounding, the exponentials and factors
    rel = off + one[:, None] + (spread * 8 + 64) * U + (0.0 if dtype == F32 else 2.0 ** -11)
    p_off = p * grow * rel * 1.01 + (0.0 if dtype == F32 else 2.0 ** -25)
    # at the target: from the f32 log probability
    lt = (zt - lse)
    t_off = p[at, y] * (2 * one + FEW * U) * grow[:, 0] + FEW * U * (dz[at, y] / dl.where(dl != 0, torch.ones_like(dl))).abs()
    p_off[at, y] = t_off + (2 * z_loss * one) * p[at, y]
    dz_off = p_off * dl.abs()[:, None] + KEPT[dtype] * dz.abs() * 1.01 + 2 * z_loss * one[:, None] * p * dl.abs()[:, None]
    if dtype != BF16 and len(rows):
        dz_off = dz_off + 2.0 ** -38 * (dl.abs()[:, None] * grow.abs().clamp_min(1)).max()
    more = 3 * 2.0 ** -22 if dtype == F32 else 0.0
    deep = 3 if dtype == F32 else 1
    dh = torch.zeros(hidden.shape, dtype=torch.float64, device=z.device)
    dh_off = dh.clone()
    dh[rows] = torch.matmul(dz, w)
    dh_off[rows] = torch.matmul(dz_off + ((vocab + 80) * U * deep + more) * dz.abs(), w.abs())
    dw = torch.matmul(dz.t().contiguous(), h)
    dw_off = torch.matmul((dz_off + ((len(rows) + 80) * U * deep + more) * dz.abs()).t().contiguous(), h.abs())
    if dtype == F32 and len(rows):
        dh_off[rows] += 2.0 ** -38 * w.abs().max() * dz.abs().sum(1, keepdim=True)
        dw_off += 2.0 ** -38 * h.abs().max() * dz.abs().sum(0)[:, None]
    return (loss, loss_off), (dh, dh_off), (dw, dw_off)


def near(got, ref, what):
    value, off = ref
    assert got.shape == value.shape, what
    g = got.double()
    bound = HALF_ULP[got.dtype] * (value.abs() + off) * 1.01 + TINY[got.dtype] + off
    fine = (g - value).abs() <= bound
    if not fine.all():
        at = tuple(torch.nonzero(~fine)[0].tolist())
        raise AssertionError(f"{what}: at {at} got {g[at].item()}, expected {value[at].item()}, bound {bound[at].item():.3g}; "
                             f"{int((~fine).sum())} of {fine.numel()} off")


def check(hidden, weight, targets, dloss, z_loss=0.0, ignore=-100):
    loss, dh, dw = reference(hidden, weight, targets, dloss, z_loss, ignore)
    near(rf().linear_cross_entropy(hidden, weight, targets, ignore_index=ignore, z_loss=z_loss), loss, "loss alone")
    got = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss, ignore_index=ignore, z_loss=z_loss)
    assert got.hidden.dtype == hidden.dtype and got.weight.dtype == weight.dtype and got.loss.dtype == F32
    near(got.loss, loss, "loss")
    near(got.hidden, dh, "dhidden")
    near(got.weight, dw, "dweight")
    assert not got.hidden[targets == ignore].any()
    return got


SIZES = [(1, 1, 1), (1, 2, 5), (2, 63, 8), (3, 64, 64), (5, 65, 72), (17, 127, 63), (63, 129, 65), (64, 640, 128),
         (65, 1000, 200), (130, 255, 301), (257, 513, 320), (300, 2049, 96), (1025, 300, 40), (40, 9001, 136)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(size, dtype):
    check(*make(*size, dtype, seed=sum(size)))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("masked", [0.3, 0.97])
def test_masked_and_z_loss(masked, kind, dtype):
    check(*make(201, 777, 160, dtype, seed=3, masked=masked, ignore=7, kind=kind), z_loss=0.01, ignore=7)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_what_lies_in_ignored_rows_reaches_nothing(dtype):
    hidden, weight, targets, dloss = make(70, 300, 72, dtype, seed=5, masked=0.4)
    clean = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    for junk in (math.nan, math.inf, -math.inf, torch.finfo(dtype).max):
        bad, bad_dloss = hidden.clone(), dloss.clone()
        bad[targets == -100] = junk
        bad_dloss[targets == -100] = junk
        got = rf().linear_cross_entropy_grad(bad, weight, targets, bad_dloss)
        for x, y in zip(got, clean):
            assert torch.equal(x, y)
        assert torch.equal(rf().linear_cross_entropy(bad, weight, targets), clean.loss)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_tokens(dtype):
    hidden, weight, _, _ = make(9, 130, 40, dtype)
    for rows, targets in ((hidden, torch.full((9,), -100, device="cuda")),
                          (hidden[:0], torch.zeros(0, dtype=torch.int64, device="cuda"))):
        got = rf().linear_cross_entropy_grad(rows, weight, targets, torch.ones(len(rows), device="cuda"))
        assert got.hidden.shape == rows.shape
        assert not got.loss.any() and not got.hidden.any() and not got.weight.any()
        assert not rf().linear_cross_entropy(rows, weight, targets).any()
        assert rf().linear_cross_entropy(rows, weight, targets, reduction="mean").isnan()
        assert rf().linear_cross_entropy(rows, weight, targets, reduction="sum").item() == 0.0
        got = rf().linear_cross_entropy_grad(rows, weight, targets, reduction="mean")
        assert got.loss.isnan() and not got.hidden.any() and not got.weight.any()


def test_targets_out_of_range_are_nan():
    hidden, weight, targets, dloss = make(40, 150, 64, BF16, seed=9)
    fine = rf().linear_cross_entropy(hidden, weight, targets)
    for wrong in (150, -1, 2 ** 31, -2 ** 40, 2 ** 62):
        bad = targets.clone()
        bad[7] = wrong
        loss = rf().linear_cross_entropy(hidden, weight, bad)
        assert loss[7].isnan()
        loss[7] = fine[7]
        assert torch.equal(loss, fine)
        got = rf().linear_cross_entropy_grad(hidden, weight, bad, dloss)
        assert got.loss[7].isnan() and got.hidden[7].isnan().all() and got.weight.isnan().all()
        assert got.hidden[torch.arange(40, device="cuda") != 7].isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_layouts(dtype):
    hidden, weight, targets, dloss = make(66, 203, 80, dtype, seed=11, masked=0.2)
    ref = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)

    def same(h, w, t, d):
        got = rf().linear_cross_entropy_grad(h, w, t, d)
        assert torch.equal(got.loss.reshape(-1), ref.loss)
        assert torch.equal(got.hidden.reshape(66, 80), ref.hidden)
        assert torch.equal(got.weight, ref.weight)

    wide = torch.full((66, 97), math.nan, dtype=dtype, device="cuda")
    wide[:, 5:85] = hidden
    same(wide[:, 5:85], weight, targets, dloss)
    tall = torch.full((203, 91), math.nan, dtype=dtype, device="cuda")
    tall[:, 3:83] = weight
    same(hidden, tall[:, 3:83], targets, dloss)
    same(hidden.t().contiguous().t(), weight.t().contiguous().t(), targets, dloss)
    same(hidden.view(6, 11, 80), weight, targets.view(6, 11), dloss.view(6, 11))
    twice = torch.stack((targets, targets), 1)
    same(hidden, torch.nn.Parameter(weight), twice[:, 0], torch.stack((dloss, dloss), 1)[:, 1])
    buffer = torch.empty(66 * 80 + 1, dtype=dtype, device="cuda")
    buffer[1:] = hidden.reshape(-1)
    same(buffer[1:].view(66, 80), weight, targets, dloss)
    # one row for all tokens
    one = rf().linear_cross_entropy_grad(hidden[:1].expand(66, 80), weight, targets, dloss)
    check(hidden[:1].expand(66, 80).contiguous(), weight, targets, dloss)
    assert one.hidden.shape == (66, 80)
    # one token, no dimension of tokens
    got = rf().linear_cross_entropy(hidden[3], weight, targets[3])
    assert got.shape == () and got == ref.loss[3]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("logit", [1e-3, 30.0, 1000.0])
def test_small_and_large_logits(logit, dtype):
    check(*make(50, 400, 64, dtype, seed=13, logit=logit))


def test_confident_tokens_keep_their_gradients():
    """Probabilities next to one: dz at the target is a difference of nearly equal numbers."""
    hidden, weight, targets, dloss = make(64, 500, 64, F32, seed=17)
    hidden = (hidden + 12.0 * weight[targets] / weight[targets].square().sum(1, keepdim=True)).contiguous()
    got = check(hidden, weight, targets, dloss)
    assert got.loss.min() < 0.02
    hidden, weight = hidden.to(BF16), weight.to(BF16)
    check(hidden, weight, targets, dloss)


def test_infinite_logits():
    hidden, weight, targets, dloss = make(6, 90, 8, F32, seed=19)
    weight[11] = 0.0
    weight[11, 0] = -math.inf
    hidden[:, 0] = hidden[:, 0].abs() + 0.1
    hidden[2, 0] = -1.0  # its logit 11 is +inf
    targets[:] = 3
    loss = rf().linear_cross_entropy(hidden, weight, targets)
    keep = torch.arange(90, device="cuda") != 11
    ref = rf().linear_cross_entropy(hidden, weight[keep].contiguous(), targets)
    assert loss[2].isnan()
    other = torch.arange(6, device="cuda") != 2
    # f32's split parts: 0 times an infinity is NaN in its low part, as the logit itself is in a product of halves
    assert (loss[other].isnan() | torch.isclose(loss[other], ref[other], rtol=1e-5)).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_reductions(dtype):
    hidden, weight, targets, _ = make(1500, 333, 48, dtype, seed=23, masked=0.3)
    loss = rf().linear_cross_entropy(hidden, weight, targets, z_loss=1e-3)
    count = int((targets != -100).sum())
    for reduction, ref, each in (("sum", loss.double().sum(), 1.0), ("mean", loss.double().sum() / count, 1.0 / count)):
        got = rf().linear_cross_entropy(hidden, weight, targets, z_loss=1e-3, reduction=reduction)
        assert got.shape == () and abs(got.item() - ref.item()) <= 2 * U * abs(ref.item())
        a = rf().linear_cross_entropy_grad(hidden, weight, targets, z_loss=1e-3, reduction=reduction)
        b = rf().linear_cross_entropy_grad(hidden, weight, targets, torch.full_like(loss, each), z_loss=1e-3)
        assert torch.equal(a.loss, got)
        for x, y in ((a.hidden, b.hidden), (a.weight, b.weight)):  # 1 / count may differ by an ulp
            assert ((x.double() - y.double()).abs() <= 2 * HALF_ULP[dtype] * y.double().abs() + TINY[dtype] + 4 * U * y.abs().max()).all()


@pytest.mark.parametrize("dtype,tokens,hidden", [(BF16, 1537, 16), (F32, 600, 9)])
def test_several_pieces_of_tokens(dtype, tokens, hidden):
    """A vocabulary of 2^20: 1024 tokens' exponentials at a time in 16 bits, 256 in f32."""
    h, w, targets, dloss = make(tokens, 1 << 20, hidden, dtype, seed=29, masked=0.1)
    got = rf().linear_cross_entropy_grad(h, w, targets, dloss, z_loss=1e-4)
    on = targets != -100
    rows = torch.nonzero(on)[:, 0]
    loss, dh, dw = torch.zeros(tokens, dtype=torch.float64, device="cuda"), torch.zeros_like(h, dtype=torch.float64), torch.zeros_like(w, dtype=torch.float64)
    for at in rows.split(256):
        z = product(h[at].double(), w.double())
        lse = torch.logsumexp(z, 1, keepdim=True)
        mine = torch.arange(len(at), device="cuda")
        loss[at] = (lse[:, 0] - z[mine, targets[at]]) + 1e-4 * lse[:, 0] ** 2
        p = torch.exp(z - lse) * (1 + 2e-4 * lse)
        p[mine, targets[at]] -= 1
        p *= dloss[at].double()[:, None]
        dh[at] = torch.matmul(p, w.double())
        dw += torch.matmul(p.t().contiguous(), h[at].double())
    tol = 2 * HALF_ULP[dtype] if dtype == BF16 else 2e-5  # dz and the result are rounded once each
    for x, y, bound in ((got.loss, loss, 1e-5), (got.hidden, dh, tol), (got.weight, dw, tol)):
        assert ((x.double() - y).norm() / y.norm()).item() < bound
    assert torch.equal(got.loss, rf().linear_cross_entropy(h, w, targets, z_loss=1e-4))


def test_offsets_past_32_bits():
    """weight has more than 2^31 elements."""
    vocab, n = 1 << 20, 2112
    gen = torch.Generator(device="cuda")
    gen.manual_seed(31)
    weight = torch.empty(vocab, n, dtype=BF16, device="cuda")
    for part in weight.split(1 << 17):
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * 0.02)
    hidden = torch.randn(3, n, generator=gen, device="cuda").to(BF16)
    targets = torch.tensor([vocab - 1, 5, vocab - 70000], device="cuda")
    dloss = torch.ones(3, device="cuda")
    z = torch.cat([product(hidden.double(), part.double()) for part in weight.split(1 << 17)], 1)
    lse = torch.logsumexp(z, 1)
    loss = lse - z[torch.arange(3, device="cuda"), targets]
    got = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    assert torch.allclose(got.loss.double(), loss, rtol=1e-5)
    p = torch.exp(z - lse[:, None])
    p[torch.arange(3, device="cuda"), targets] -= 1
    for at in (0, 5, vocab // 2, vocab - 70000, vocab - 1):
        ref = p[:, at] @ hidden.double()
        assert ((got.weight[at].double() - ref).norm() / ref.norm()).item() < 2.0 ** -7
    dh = sum(torch.matmul(p[:, i: i + (1 << 17)].contiguous(), weight[i: i + (1 << 17)].double()) for i in range(0, vocab, 1 << 17))
    assert ((got.hidden.double() - dh).norm() / dh.norm()).item() < 2.0 ** -7


def test_equal_inputs_give_equal_bits():
    for args in (make(300, 5000, 136, BF16, seed=37), make(3, 9000, 512, F32, seed=38)):
        a = rf().linear_cross_entropy_grad(*args)
        for _ in range(3):
            for x, y in zip(rf().linear_cross_entropy_grad(*args), a):
                assert torch.equal(x, y)


def test_another_stream():
    args = make(257, 1000, 72, BF16, seed=41)
    ref = rf().linear_cross_entropy_grad(*args)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = rf().linear_cross_entropy_grad(*args)
    stream.synchronize()
    for x, y in zip(got, ref):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_captured_and_replayed(dtype):
    hidden, weight, targets, dloss = make(130, 700, 64, dtype, seed=43, masked=0.2)
    rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rf().linear_cross_entropy_grad(hidden, weight, targets, dloss)
        mean = rf().linear_cross_entropy(hidden, weight, targets, reduction="mean")
    for turn in range(4):
        h2, w2, t2, d2 = make(130, 700, 64, dtype, seed=100 + turn, masked=0.1 * turn)
        for x, y in ((hidden, h2), (weight, w2), (targets, t2), (dloss, d2)):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        ref = rf().linear_cross_entropy_grad(h2, w2, t2, d2)
        for x, y in zip(got, ref):
            assert torch.equal(x, y), turn
        assert torch.equal(mean, rf().linear_cross_entropy(h2, w2, t2, reduction="mean"))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,vocab,n", [(60, 16000, 576), (65, 8200, 1024), (150, 20011, 256), (193, 4100, 2048),
                                            (520, 3000, 70), (300, 33000, 128)])
@pytest.mark.parametrize("masked", [0.0, 0.6, 0.98])
def test_few_tokens_of_larger_tables(masked, tokens, vocab, n, dtype):
    """Tiles of every width, whole and split, with as many tokens as the call has or far fewer."""
    check(*make(tokens, vocab, n, dtype, seed=vocab, masked=masked))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_that_share_memory(dtype):
    """Expanded rows are read in place; the gradients are those of rows apart."""
    hidden, weight, targets, dloss = make(70, 300, 128, dtype, seed=9, masked=0.2)
    one = hidden[3:4].expand(70, 128)
    check(one, weight, targets, dloss)
    same = weight[5:6].expand(300, 128)
    check(hidden, same, targets, dloss)
    rows = weight.as_strided((200, 128), (64, 1))  # each row begins in the middle of the one before
    check(hidden, rows, targets % 200, dloss)
    # one tensor as both: a table of 64 rows against itself
    check(weight[:64], weight[:64], targets[:64].clamp(min=0) % 64, dloss[:64])
