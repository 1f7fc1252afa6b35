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
