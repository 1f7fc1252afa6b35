"""The residual-block operators against their definitions in 64 bits.

Tolerances are bounds on f32 arithmetic, stated before any run.  U is half an
f32 ulp, 2^-24.  An output is rounded once to its dtype (half an ulp: 2^-8,
2^-11 or U of its value, plus the subnormal spacing of float16).  Behind that:
- a row mean is a sum over at most 16 terms a lane, 6 steps of a wave and 8
  waves, and its terms carry a few roundings: DEEP * U of the sum of the terms'
  magnitudes covers it;
- a sum over rows adds at most rows terms in sequence: (rows + DEEP) * U of the
  magnitudes;
- sigmoid, exp and erf of the device are within FEW ulps, exp(x) within |x| U
  more for the product with log2(e).
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEEP = 64
FEW = 16
HALF_ULP = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
PAIRS = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)]


def rf():
    import rollfast_amd

    return rollfast_amd


def rand(shape, dtype, seed, scale=1.0, mean=0.0):
    gen = torch.Generator()
    gen.manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale + mean).to(dtype).cuda()


def d(x):
    return None if x is None else x.detach().double().cpu()


def close(got, ref, slack, what):
    """|got - ref| within the rounding to got's dtype and `slack`."""
    dtype = got.dtype
    g, slack = d(got), torch.as_tensor(slack, dtype=torch.float64).expand(ref.shape)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), what
    bound = HALF_ULP[dtype] * (ref.abs() + slack) * 1.01 + TINY[dtype] + slack
    off = (g - ref).abs()
    fine = (off <= bound) | torch.isnan(ref) | (g == ref.to(dtype).double())  # past the largest value: Inf
    if not fine.all():
        at = torch.nonzero(~fine)[0].tolist()
        i = tuple(at)
        raise AssertionError(f"{what}: at {i} got {g[i].item()}, expected {ref[i].item()}, off {off[i].item():.3g}, "
                             f"bound {bound[i].item():.3g}; {int((~fine).sum())} of {fine.numel()} off")


def encode(x):
    """(codes, exponents) of the definition, on x [rows, cols] in 64 bits."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.zeros(rows, blocks * 32, dtype=torch.float64)
    v[:, :cols] = x.double().cpu()
    v = v.view(rows, blocks, 32)
    top = v.abs().amax(2)
    _, power = torch.frexp(top)
    e = torch.where(top > 0, (power - 1 + 127 - 6).clamp_min(1), torch.ones_like(power))
    e = torch.where(torch.isfinite(top), e, torch.full_like(e, 255))
    codes = torch.round(torch.nan_to_num(v, 0, 0, 0) / torch.exp2(e.double() - 127)[..., None]).clamp(-127, 127)
    codes[e == 255] = 0
    return codes.to(torch.int8).view(rows, -1), e.to(torch.uint8)


def decode(codes, e, cols):
    step = torch.exp2(e.double() - 127)
    step[e == 255] = math.nan
    return (codes.view(*e.shape, 32).double() * step[..., None]).reshape(codes.shape)[:, :cols]


def kept(x):
    return decode(*encode(x), x.shape[1])


def check_codes(ck, x, what):
    codes, e = encode(x)
    assert torch.equal(ck.exponents.cpu().view(e.shape), e), what
    assert torch.equal(ck.codes.cpu().view(codes.shape), codes), what


# ------------------------------------------------------------- checkpoints ---
SHAPES = [(1, 1), (3, 7), (5, 31), (4, 32), (7, 33), (2, 64), (70, 301), (130, 768), (9, 1031), (33, 4096), (6, 8200),
          (2, 16411)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_checkpoint_round_trip(shape, dtype):
    x = rand(shape, dtype, 1)
    x = x * torch.exp2(torch.randint(-20, 10, (shape[0], 1), generator=torch.Generator().manual_seed(2)).cuda()).to(dtype)
    ck = rf().checkpoint_activations(x)
    check_codes(ck, x, "codes")
    for out in (None, F32, BF16, F16):
        got = rf().restore_activations(ck, dtype=out)
        assert got.dtype == (out or dtype) and got.shape == x.shape
        assert torch.equal(got.cpu(), kept(x).to(got.dtype)), out


def test_checkpoint_extremes():
    """Zeros, subnormals, the largest values, saturation at 127.5 steps, ties,
    and blocks that are not finite beside ones that are."""
    x = torch.zeros(12, 96)
    x[0, 3] = 1.0
    x[1] = 2.0 ** -149
    x[2, :40] = torch.linspace(-1, 1, 40) * 2.0 ** -126
    x[3] = torch.finfo(F32).max
    x[4, 0], x[4, 1], x[4, 33] = 127.75, -127.5, 64.0
    x[5, :32] = torch.arange(32) + 0.5 + 64
    x[6, 5] = math.inf
    x[7, 40] = -math.inf
    x[8, 95] = math.nan
    x[9] = -torch.finfo(F32).max
    x[10, 0], x[10, 1] = 2.0 ** 127, -1.0
    x[11, 0], x[11, 1] = -0.0, 2.0 ** -120
    x = x.cuda()
    ck = rf().checkpoint_activations(x)
    check_codes(ck, x, "codes")
    got, ref = rf().restore_activations(ck).double().cpu(), kept(x)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(ref))
    assert torch.isnan(got[6, :32]).all() and torch.isfinite(got[6, 32:]).all()


def test_checkpoint_strides_and_offsets():
    base = rand((40, 3, 330), BF16, 3)
    for x in (base[:, 1], base[:, :, 5:306], base[::2, 2, 1:], base[..., 0:1], base.transpose(0, 1),
              base[0].t(), base[:1].expand(4, 3, 330), base[0, 0], base.permute(2, 0, 1)):
        ck = rf().checkpoint_activations(x)
        flat = x.contiguous().view(-1, x.shape[-1])
        check_codes(ck, flat, x.shape)
        assert torch.equal(rf().restore_activations(ck), rf().restore_activations(rf().checkpoint_activations(flat)).view(x.shape))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_checkpoint_of_nothing(dtype):
    ck = rf().checkpoint_activations(torch.empty(0, 5, 33, dtype=dtype, device="cuda"))
    assert rf().restore_activations(ck).shape == (0, 5, 33)


# ------------------------------------------------------------ weight grads ---
def wgrad_case(t, n, k, dtype, out, seed=5):
    dy, x = rand((t, n), dtype, seed, 1e-2), rand((t, k), F32, seed + 1)
    ck = rf().checkpoint_activations(x)
    got = rf().linear_weight_grad(dy, ck, dtype=out)
    x8 = decode(ck.codes.cpu(), ck.exponents.cpu(), k)
    ref = d(dy).t() @ x8
    # products are exact; f32 sums in some order: t terms in sequence at most
    close(got, ref, (t + 8) * U * (d(dy).abs().t() @ x8.abs()), (t, n, k, dtype, out))


@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("t,n,k", [(1, 1, 1), (1, 64, 64), (2, 7, 33), (31, 40, 65), (33, 129, 127), (64, 256, 256),
                                   (65, 257, 300), (100, 517, 301), (257, 96, 544), (511, 130, 40), (1000, 33, 31)])
def test_weight_grad(t, n, k, dtype, out):
    wgrad_case(t, n, k, dtype, out)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("t,n,k", [(5000, 64, 96), (2049, 768, 320), (4100, 1, 1), (300, 1100, 1030)])
def test_weight_grad_long_sums_and_many_tiles(t, n, k, dtype):
    wgrad_case(t, n, k, dtype, F32)


@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F32, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("t,n,k", [(1, 9, 35), (70, 140, 260), (3000, 65, 70)])
def test_weight_grad_accumulates(t, n, k, dtype, out):
    dy, x = rand((t, n), dtype, 7, 1e-2), rand((t, k), BF16, 8)
    acc = rand((n, k), out, 9, 0.1)
    ck = rf().checkpoint_activations(x)
    ref = d(dy).t() @ kept(x) + d(acc)
    slack = (t + 8) * U * (d(dy).abs().t() @ kept(x).abs()) + 2 * U * d(acc).abs()
    same = rf().linear_weight_grad(dy, ck, out=acc, accumulate=True)
    assert same is acc
    close(acc, ref, slack, "accumulated")
    rf().linear_weight_grad(dy, ck, out=acc)
    close(acc, d(dy).t() @ kept(x), slack, "overwritten")


@pytest.mark.parametrize("t,n,k", [(32, 4096, 4096), (333, 4096, 4096), (290, 4104, 3936), (64, 3969, 4100), (450, 4098, 4001)])
def test_weight_grad_large_tiles(t, n, k):
    """Enough outputs for the largest tiles: rows of whole 16-byte units and
    others, tails of rows, columns and outputs; strided and offset rows."""
    wgrad_case(t, n, k, BF16, F32)
    x = rand((t, k), BF16, 11)
    ck = rf().checkpoint_activations(x)
    base = rand((t, n + 24), BF16, 12, 1e-2)
    for off in (8, 3):
        dy = base[:, off: off + n]
        a, b = d(dy), kept(x)
        close(rf().linear_weight_grad(dy, ck, dtype=F32), a.t() @ b, (t + 8) * U * (a.abs().t() @ b.abs()), (t, n, k, off))


def test_weight_grad_large_tiles_are_those_of_the_small():
    """The sums of a column do not depend on the tile but for their order: an
    Inf and a NaN reach their rows of outputs and nothing else."""
    t, n, k = 300, 4096, 4096
    dy, x = rand((t, n), BF16, 1, 1e-2), rand((t, k), BF16, 2)
    dy[299, 7], dy[5, 4000] = math.inf, math.nan
    x[:, 0] = x[:, 0].abs() + 0.5
    got = rf().linear_weight_grad(dy, rf().checkpoint_activations(x), dtype=F32)
    assert not torch.isfinite(got[7, 0]) and torch.isnan(got[4000]).all()
    mask = torch.ones(n, dtype=torch.bool)
    mask[[7, 4000]] = False
    assert torch.isfinite(got.cpu()[mask]).all()
    small = rf().linear_weight_grad(dy[:, 64:192].contiguous(), rf().checkpoint_activations(x), dtype=F32)
    assert (got[64:192] - small).abs().max() <= 2 * (t + 8) * U * (d(dy[:, 64:192]).abs().t() @ kept(x).abs()).max()


def test_weight_grad_of_no_rows():
    ck = rf().checkpoint_activations(torch.empty(0, 40, device="cuda"))
    dy = torch.empty(0, 9, device="cuda", dtype=BF16)
    assert torch.equal(rf().linear_weight_grad(dy, ck), torch.zeros(9, 40, device="cuda", dtype=BF16))
    acc = rand((9, 40), F32, 1)
    before = acc.clone()
    rf().linear_weight_grad(dy, ck, out=acc, accumulate=True)
    assert torch.equal(acc, before)


def test_weight_grad_strided_gradient():
    """dy with a row stride, at an odd offset, broadcast and transposed."""
    x = rand((6, 20, 70), BF16, 3)
    ck = rf().checkpoint_activations(x)
    base = rand((6, 20, 301), BF16, 4, 1e-2)
    one = rand((1, 1, 50), BF16, 5)
    for dy in (base[..., 1:97], base[..., 3:4], one.expand(6, 20, 50), rand((50, 20, 6), BF16, 6).permute(2, 1, 0)):
        got = rf().linear_weight_grad(dy, ck, dtype=F32)
        a, b = d(dy.contiguous()).view(120, -1), kept(x.view(120, 70))
        close(got, a.t() @ b, 128 * U * (a.abs().t() @ b.abs()), tuple(dy.shape))


def test_weight_grad_extreme_values():
    """Large and tiny magnitudes of f32 gradients keep their f32 accuracy;
    an Inf or NaN reaches exactly its row and column of outputs."""
    t, n, k = 40, 70, 64
    dy = rand((t, n), F32, 1)
    dy[:, 3] *= 1e30
    dy[:, 4] *= 1e-30
    dy[0, 5] = 3e38
    x = rand((t, k), F32, 2)
    ck = rf().checkpoint_activations(x)
    a, b = d(dy), kept(x)
    close(rf().linear_weight_grad(dy, ck), a.t() @ b, (t + 8) * U * (a.abs().t() @ b.abs()), "wide range")
    dy = rand((t, n), F32, 1)
    dy[7, 2], dy[9, 11] = math.inf, math.nan
    x[:, 0] = x[:, 0].abs() + 0.5  # no zero codes in column 0
    ck = rf().checkpoint_activations(x)
    for dtype in (F32, BF16, F16):
        got = rf().linear_weight_grad(dy.to(dtype), ck, dtype=F32)
        assert not torch.isfinite(got[2, 0]) and torch.isnan(got[11]).all()
        mask = torch.ones(n, dtype=torch.bool)
        mask[[2, 11]] = False
        assert torch.isfinite(got.cpu()[mask]).all(), dtype
    x[3, 40] = math.nan  # the block of columns 32 .. 63 reads back NaN
    got = rf().linear_weight_grad(rand((t, n), BF16, 1), rf().checkpoint_activations(x))
    assert torch.isnan(got[:, 32:64]).all() and torch.isfinite(got[:, :32]).all()


# ------------------------------------------------------- gated activation ---
def act64(x, name):
    if name == "silu":
        s = torch.sigmoid(x)
        return x * s, s * (1 + x * (1 - s))
    if name == "gelu":
        p = 0.5 * torch.erfc(-x / math.sqrt(2))
        return x * p, p + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (x + 0.044715 * x ** 3))
    return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 3 * 0.044715 * x * x)


def act_slack(x):
    """Error of the activation and of its slope over |x| and over 1."""
    return (FEW + x.abs().clamp_max(100.0)) * U * x.abs(), (FEW + x.abs().clamp_max(100.0)) * U * (1 + x.abs().clamp_max(8.0))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (64, 301), (17, 2048), (2, 11008)])
@pytest.mark.parametrize("save", ["int8", "input"])
def test_gated(shape, name, dtype, save):
    g, u, dh = rand(shape, dtype, 1, 2.0), rand(shape, dtype, 2), rand(shape, dtype, 3, 1e-2)
    h, saved = rf().gated_activation(g, u, activation=name, save=save, checkpoint_output=True)
    a, _ = act64(d(g), name)
    close(h, a * d(u), act_slack(d(g))[0] * d(u).abs() * 2, "h")
    check_codes(saved.output, h, "checkpoint of h")
    dg, du = rf().gated_activation_grad(dh, saved)
    x, y = (kept(g), kept(u)) if save == "int8" else (d(g), d(u))
    a, slope = act64(x, name)
    sa, ss = act_slack(x)
    close(dg, d(dh) * y * slope, 2 * (d(dh) * y).abs() * ss, "dgate")
    close(du, d(dh) * a, 2 * d(dh).abs() * sa, "dup")
    plain, none = rf().gated_activation(g, u, activation=name, save=None)
    assert none is None and torch.equal(plain, h)


@pytest.mark.parametrize("cols", [1, 31, 32, 100, 512])
def test_gated_fused_halves(cols):
    """One tensor with both halves gives the bits of the two-tensor form."""
    gu, dh = rand((3, 9, 2 * cols), BF16, 1), rand((3, 9, cols), BF16, 2)
    for save in ("int8", "input"):
        h, saved = rf().gated_activation(gu, save=save)
        h2, saved2 = rf().gated_activation(gu[..., :cols], gu[..., cols:], save=save)
        assert torch.equal(h, h2)
        both = rf().gated_activation_grad(dh, saved)
        dg, du = rf().gated_activation_grad(dh, saved2)
        assert both.shape == gu.shape and torch.equal(both, torch.cat((dg, du), -1))


def test_gated_extremes():
    x = torch.tensor([[0.0, -0.0, 90.0, -90.0, 1e30, -1e30, 200.0, -200.0, math.nan]], device="cuda")
    for name in ("silu", "gelu", "gelu_tanh"):
        h, saved = rf().gated_activation(x, torch.ones_like(x), activation=name, save="input")
        assert torch.isnan(h[0, 8]) and torch.isfinite(h[0, :8]).all(), name
        assert (h[0, [3, 5, 7]] .abs() < 1e-30).all() and torch.equal(h[0, [2, 4, 6]], x[0, [2, 4, 6]]), name
        dg, _ = rf().gated_activation_grad(torch.ones_like(x), saved)
        assert torch.isfinite(dg[0, :4]).all() and torch.isfinite(dg[0, 6:8]).all(), name


# ------------------------------------------------------------------- norms ---
def stats64(x, norm, eps):
    mean = x.mean(1, keepdim=True) if norm == "layer" else torch.zeros(x.shape[0], 1, dtype=torch.float64)
    if norm == "none":
        return mean, torch.ones_like(mean)
    return mean, 1 / ((x - mean).pow(2).mean(1, keepdim=True) + eps).sqrt()


def hat_slack(x, mean, rstd, norm):
    """Error of (x - mean) rstd: of the statistics and of the subtraction."""
    s = DEEP * U * ((x - mean) * rstd).abs()
    if norm == "layer":
        s = s + DEEP * U * rstd * (x.abs() + x.abs().mean(1, keepdim=True))
    return s


def norm_back64(g, xhat, rstd, norm):
    if norm == "none":
        return g
    out = g - xhat * (g * xhat).mean(1, keepdim=True)
    if norm == "layer":
        out = out - g.mean(1, keepdim=True)
    return rstd * out


def back_slack(g, xhat, rstd, sx):
    """Error of norm_back: relative to its terms' magnitudes, and sx, the
    error of xhat, through both places where it enters."""
    m = (g * xhat).abs().mean(1, keepdim=True)
    ms = (g.abs() * sx).mean(1, keepdim=True)
    return rstd * (2 * DEEP * U * (g.abs() + g.abs().mean(1, keepdim=True) + xhat.abs() * m) + sx * m + xhat.abs() * ms)


def check_prenorm(rows, cols, x_dtype, y_dtype, norm, w_dtype, save, bias, dres, seed=1, strided=False):
    width = cols + 13 if strided else cols
    x = rand((rows, width), x_dtype, seed, 1.0, 0.3)[:, width - cols:]
    w = None if w_dtype is None else rand((cols,), w_dtype, seed + 1, 0.2, 1.0)
    b = rand((cols,), w_dtype or F32, seed + 2, 0.2) if bias else None
    dy = rand((rows, width), y_dtype, seed + 3, 1e-2)[:, :cols]
    dr = rand((rows, cols), x_dtype, seed + 4, 1e-2) if dres else None
    eps = 1e-5
    y, saved = rf().prenorm(x, w, b, norm=norm, eps=eps, dtype=y_dtype, save=save, checkpoint_output=True)
    x6, w6, b6 = d(x), 1.0 if w is None else d(w), 0.0 if b is None else d(b)
    mean, rstd = stats64(x6, norm, eps)
    hat, sh = (x6 - mean) * rstd, hat_slack(x6, mean, rstd, norm)
    ww = torch.ones(cols, dtype=torch.float64) * w6
    close(y, hat * ww + b6, sh * ww.abs() + 4 * U * ((hat * ww).abs() + torch.as_tensor(b6).abs()), "y")
    check_codes(saved.output, y, "checkpoint of y")
    got = rf().prenorm_grad(dy, saved, dresidual=dr)
    xs = kept(x) if save == "int8" else x6
    hat, sh = (xs - mean) * rstd, hat_slack(xs, mean, rstd, norm) + hat_slack(x6, mean, rstd, norm)
    g = d(dy) * ww
    ref = norm_back64(g, hat, rstd, norm) + (0.0 if dr is None else d(dr))
    close(got.x, ref, back_slack(g, hat, rstd, sh) + (0.0 if dr is None else 4 * U * d(dr).abs()), "dx")
    terms = (d(dy) * hat).abs().sum(0)
    if w is None:
        assert got.weight is None
    else:
        close(got.weight, (d(dy) * hat).sum(0), (rows + DEEP) * U * terms + (d(dy).abs() * sh).sum(0), "dweight")
    if b is None:
        assert got.bias is None
    else:
        close(got.bias, d(dy).sum(0), (rows + DEEP) * U * d(dy).abs().sum(0), "dbias")
    again = rf().prenorm_grad(dy, saved, dresidual=dr)
    assert all((p is None and q is None) or torch.equal(p, q) for p, q in zip(got, again)), "runs differ"
    plain, none = rf().prenorm(x, w, b, norm=norm, eps=eps, dtype=y_dtype, save=None)
    assert none is None and torch.equal(plain, y)


NORM_SHAPES = [(1, 1), (3, 7), (5, 32), (70, 301), (300, 768), (9, 1024), (7, 1031), (20, 2048), (6, 2056), (19, 4096),
               (5, 4100), (4, 8192), (3, 8200), (2, 16411)]


@pytest.mark.parametrize("x_dtype,y_dtype", PAIRS)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("save", ["int8", "input"])
def test_prenorm(rows, cols, x_dtype, y_dtype, norm, save):
    check_prenorm(rows, cols, x_dtype, y_dtype, norm, F32, save, norm == "layer", True)


@pytest.mark.parametrize("w_dtype", [None, BF16, F16])
@pytest.mark.parametrize("norm,bias", [("rms", False), ("rms", True), ("layer", False)])
def test_prenorm_vectors(w_dtype, norm, bias):
    for rows, cols in ((40, 130), (11, 3000), (3, 9000)):
        check_prenorm(rows, cols, BF16, BF16, norm, w_dtype, "int8", bias, False)
        check_prenorm(rows, cols, F32, BF16, norm, w_dtype, "input", bias, True, strided=True)


def check_postnorm(shape, r_dtype, u_dtype, norm, gates, follows, save, vectors=F32, seed=1, dout_given=True, bias=None):
    """gates: None, 'one', or the number of leading dimensions the gate varies over."""
    cols, rows = shape[-1], math.prod(shape[:-1])
    bias = norm == "layer" if bias is None else bias
    r, u = rand(shape, r_dtype, seed), rand(shape, u_dtype, seed + 1, 0.5, 0.1)
    w = None if norm == "none" else rand((cols,), vectors, seed + 2, 0.2, 1.0)
    b = rand((cols,), vectors, seed + 3, 0.2) if bias and norm != "none" else None
    gate_shape = None if gates is None else (cols,) if gates == "one" else (
        *shape[:gates], *([1] * (len(shape) - 1 - gates)), cols)
    gate = None if gate_shape is None else rand(gate_shape, vectors, seed + 4, 0.2, 0.4)
    w2 = rand((cols,), vectors, seed + 5, 0.2, 1.0) if follows else None
    b2 = rand((cols,), vectors, seed + 6, 0.2) if follows and bias else None
    dout = rand(shape, r_dtype, seed + 7, 1e-2) if dout_given else None
    dy = rand(shape, u_dtype, seed + 8, 1e-2) if follows else None
    eps, s, a = 1e-5, 0.7, 1.25
    out, y, saved = rf().postnorm_residual(r, u, w, b, gate, norm=norm, eps=eps, branch_scale=s, residual_scale=a,
                                           next_norm=(follows or None), next_weight=w2, next_bias=b2, next_eps=eps,
                                           save=save, checkpoint_output=bool(follows))
    f = lambda t: d(t).reshape(rows, cols)  # noqa: E731
    r6, u6 = f(r), f(u)
    one = torch.ones(cols, dtype=torch.float64)
    w6, b6 = one if w is None else d(w), 0 * one if b is None else d(b)
    g6 = one.expand(rows, cols) if gate is None else d(gate).expand(shape).reshape(rows, cols)
    mean, rstd = stats64(u6, norm, eps)
    hat, sh = (u6 - mean) * rstd, hat_slack(u6, mean, rstd, norm)
    n = hat * w6 + b6
    close(f32view(out, rows, cols), a * r6 + s * g6 * n,
          (s * g6).abs() * (sh * w6.abs() + 8 * U * ((hat * w6).abs() + b6.abs())) + 4 * U * (a * r6).abs(), "out")
    if follows:
        v6 = f(out)  # the next norm acts on the residual as it is stored
        mean2, rstd2 = stats64(v6, follows, eps)
        hat2, sh2 = (v6 - mean2) * rstd2, hat_slack(v6, mean2, rstd2, follows)
        w26, b26 = d(w2), 0 * one if b2 is None else d(b2)
        close(f32view(y, rows, cols), hat2 * w26 + b26, sh2 * w26.abs() + 4 * U * ((hat2 * w26).abs() + b26.abs()), "y")
        check_codes(saved.output, y.reshape(rows, cols), "checkpoint of y")
        if save == "int8":
            codes, e = encode(f(out))
            assert torch.equal(saved.hidden.cpu(), codes) and torch.equal(saved.hidden_exponents.cpu(), e)
    if save == "int8":
        codes, e = encode(u6)
        assert torch.equal(saved.branch.cpu(), codes) and torch.equal(saved.branch_exponents.cpu(), e)
    got = rf().postnorm_residual_grad(dout, dy, saved)
    t = torch.zeros(rows, cols, dtype=torch.float64) if dout is None else f(dout)
    st = 4 * U * t.abs()
    if follows:
        vs = kept(v6) if save == "int8" else v6
        hat2 = (vs - mean2) * rstd2
        sh2 = sh2 + hat_slack(vs, mean2, rstd2, follows)
        dy6 = f(dy)
        g2 = dy6 * w26
        t = t + norm_back64(g2, hat2, rstd2, follows)
        st = st + back_slack(g2, hat2, rstd2, sh2)
        close(got.next_weight, (dy6 * hat2).sum(0),
              (rows + DEEP) * U * (dy6 * hat2).abs().sum(0) + (dy6.abs() * sh2).sum(0), "dnext_weight")
        if b2 is not None:
            close(got.next_bias, dy6.sum(0), (rows + DEEP) * U * dy6.abs().sum(0), "dnext_bias")
    close(f32view(got.residual, rows, cols), a * t, a * st + 4 * U * (a * t).abs(), "dresidual")
    us = kept(u6) if save == "int8" else u6
    hat = (us - mean) * rstd
    sh = 0 * hat if norm == "none" else sh + hat_slack(us, mean, rstd, norm)
    gn, sgn = s * g6 * w6 * t, (s * g6 * w6).abs() * st
    back = norm_back64(gn, hat, rstd, norm)
    slack = back_slack(gn, hat, rstd, sh) + rstd * (sgn + sgn.mean(1, keepdim=True)
                                                    + hat.abs() * (sgn * hat.abs()).mean(1, keepdim=True))
    if follows:  # the row sums written out in dhidden, g2 and xhat: their parts' magnitudes
        h = (s * g6 * w6).abs()
        parts = rstd2 * (g2.abs() + g2.abs().mean(1, keepdim=True) + hat2.abs() * (g2 * hat2).abs().mean(1, keepdim=True))
        slack = slack + 2 * DEEP * U * rstd * (h * parts + (h * parts).mean(1, keepdim=True)
                                               + hat.abs() * (h * parts * hat.abs()).mean(1, keepdim=True))
    close(f32view(got.branch, rows, cols), back, slack, "dbranch")
    deep = (rows + DEEP) * U
    if w is not None:
        terms = s * g6 * hat * t
        close(got.weight, terms.sum(0), deep * terms.abs().sum(0) + (s * g6.abs() * (sh * t.abs() + hat.abs() * st)).sum(0),
              "dweight")
    if b is not None:
        close(got.bias, (s * g6 * t).sum(0), deep * (s * g6 * t).abs().sum(0) + (s * g6.abs() * st).sum(0), "dbias")
    if gate is not None:
        n = hat * w6 + b6
        terms, sterm = s * n * t, s * (n.abs() * st + sh * w6.abs() * t.abs() + 4 * U * (hat * w6 * t).abs()
                                       + 4 * U * (b6 * t).abs())
        # P and Q are summed apart
        mags = s * ((hat * w6 * t).abs() + (b6 * t).abs())
        over = lambda z: z.reshape(*shape).sum_to_size(gate_shape)  # noqa: E731
        close(got.gate, over(terms), deep * over(mags) + over(sterm), "dgate")
    again = rf().postnorm_residual_grad(dout, dy, saved)
    assert all((p is None and q is None) or torch.equal(p, q) for p, q in zip(got, again)), "runs differ"
    plain = rf().postnorm_residual(r, u, w, b, gate, norm=norm, eps=eps, branch_scale=s, residual_scale=a,
                                   next_norm=(follows or None), next_weight=w2, next_bias=b2, next_eps=eps, save=None)
    assert torch.equal(plain[0], out) and plain[2] is None and (y is None or torch.equal(plain[1], y))


def f32view(t, rows, cols):
    return t.reshape(rows, cols)


@pytest.mark.parametrize("r_dtype,u_dtype", PAIRS)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("save", ["int8", "input"])
def test_postnorm_with_next(rows, cols, r_dtype, u_dtype, norm, save):
    check_postnorm((rows, cols), r_dtype, u_dtype, norm, "one", norm, save)


@pytest.mark.parametrize("norm,follows", [("rms", None), ("layer", None), ("none", None), ("none", "rms"),
                                          ("none", "layer"), ("rms", "layer"), ("layer", "rms")])
@pytest.mark.parametrize("gates", [None, "one"])
@pytest.mark.parametrize("save", ["int8", "input"])
def test_postnorm_kinds(norm, follows, gates, save):
    for rows, cols in ((50, 130), (13, 3000), (3, 9001)):
        check_postnorm((rows, cols), BF16, BF16, norm, gates, follows, save)
        check_postnorm((rows, cols), F32, F32, norm, gates, follows, save, vectors=BF16)


@pytest.mark.parametrize("shape,vary", [((1, 5, 64), 1), ((3, 50, 130), 1), ((40, 9, 301), 1), ((3, 50, 130), 2),
                                        ((700, 3, 40), 1), ((700, 3, 40), 2), ((3, 700, 1500), 2), ((2, 3, 5, 96), 2),
                                        ((5, 64, 4096), 1), ((600, 1, 2048), 1), ((530, 2, 9000), 1), ((3, 4, 9000), 1)])
@pytest.mark.parametrize("norm,bias", [("rms", False), ("layer", True)])
def test_postnorm_gates(shape, vary, norm, bias):
    """A gate for every run of rows, from one run to a run of one row."""
    check_postnorm(shape, F32, F32, norm, vary, norm, "input", bias=bias)
    check_postnorm(shape, BF16, BF16, norm, vary, None, "int8", vectors=BF16, bias=bias)


# around the widths at which rows take more lanes, and no longer stay in registers
BROAD_SHAPES = [(11, 8193), (300, 8704), (21, 12288), (9, 16379), (13, 16384), (5, 16385), (6, 16400)]


@pytest.mark.parametrize("r_dtype,u_dtype", PAIRS)
@pytest.mark.parametrize("rows,cols", BROAD_SHAPES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("save", ["int8", "input"])
def test_broad_rows(rows, cols, r_dtype, u_dtype, norm, save):
    check_prenorm(rows, cols, r_dtype, u_dtype, norm, F32, save, norm == "layer", True)
    check_postnorm((rows, cols), r_dtype, u_dtype, norm, "one", norm, save)


@pytest.mark.parametrize("shape,vary", [((4, 31, 9000), 1), ((300, 2, 8704), 1), ((7, 1, 16384), 1), ((260, 1, 12290), 1)])
@pytest.mark.parametrize("norm,follows,bias", [("rms", "rms", False), ("layer", None, True), ("none", "layer", False)])
def test_broad_rows_gates(shape, vary, norm, follows, bias):
    check_postnorm(shape, F32, F32, norm, vary, follows, "input", bias=bias)
    check_postnorm(shape, BF16, BF16, norm, vary, follows, "int8", vectors=F16, bias=bias, dout_given=False)


@pytest.mark.parametrize("shape", [(16, 9, 70), (17, 9, 70), (32, 200, 96), (33, 40, 130), (66, 41, 391), (382, 5, 99), (255, 8, 64)])
@pytest.mark.parametrize("gate_dtype", [F32, BF16, F16])
def test_postnorm_many_gates(shape, gate_dtype):
    """Numbers of gates around those at which the final sums are dealt out otherwise."""
    check_postnorm(shape, F32, BF16, "layer", 1, "rms", "input", vectors=gate_dtype, bias=True)
    check_postnorm(shape, BF16, BF16, "rms", 1, "layer", "int8", vectors=gate_dtype)


@pytest.mark.parametrize("gates", [1, 3, 40])
def test_gates_without_rows(gates):
    r, u = torch.empty(gates, 0, 50, dtype=BF16, device="cuda"), torch.empty(gates, 0, 50, dtype=BF16, device="cuda")
    w, gate = rand((50,), F32, 1), rand((gates, 1, 50), F32, 2)
    out, y, saved = rf().postnorm_residual(r, u, w, w, gate, norm="layer", next_norm="rms", next_weight=w)
    got = rf().postnorm_residual_grad(out, y, saved)
    assert got.gate.shape == gate.shape
    for g in (got.weight, got.bias, got.gate, got.next_weight):
        assert torch.equal(g, torch.zeros_like(g))


def test_postnorm_without_dout_and_mixed_vectors():
    check_postnorm((30, 200), BF16, BF16, "rms", "one", "rms", "int8", dout_given=False)
    check_postnorm((30, 200), F32, F16, "layer", None, "layer", "input", vectors=F16, dout_given=False)


def test_postnorm_strided_rows():
    r, u = rand((12, 3, 300), BF16, 1), rand((12, 400), BF16, 2)
    args = {"next_norm": "rms", "branch_scale": 0.5}
    out, y, saved = rf().postnorm_residual(r[:, 1, 7:207], u[:, 3:203], **args)
    out2, y2, saved2 = rf().postnorm_residual(r[:, 1, 7:207].contiguous(), u[:, 3:203].contiguous(), **args)
    assert torch.equal(out, out2) and torch.equal(y, y2) and torch.equal(saved.branch, saved2.branch)
    dout, dy = rand((12, 300), BF16, 3)[:, 9:209], rand((1, 200), BF16, 4).expand(12, 200)
    for p, q in zip(rf().postnorm_residual_grad(dout, dy, saved),
                    rf().postnorm_residual_grad(dout.contiguous(), dy.contiguous(), saved2)):
        assert (p is None and q is None) or torch.equal(p, q)


def test_norms_of_no_rows():
    x = torch.empty(0, 50, device="cuda", dtype=BF16)
    w, gate = rand((50,), F32, 1), rand((50,), F32, 2)
    y, saved = rf().prenorm(x, w)
    g = rf().prenorm_grad(y, saved)
    assert g.x.shape == (0, 50) and torch.equal(g.weight, torch.zeros_like(w))
    out, y, saved = rf().postnorm_residual(x, x, w, w, gate, norm="layer", next_norm="layer", next_weight=w, next_bias=w)
    g = rf().postnorm_residual_grad(out, y, saved)
    for v in (g.weight, g.bias, g.gate, g.next_weight, g.next_bias):
        assert torch.equal(v, torch.zeros_like(w))
    empty = torch.empty(0, 4, 50, device="cuda", dtype=BF16)
    out, y, saved = rf().postnorm_residual(empty, empty, w, None, torch.empty(0, 1, 50, device="cuda"))
    assert rf().postnorm_residual_grad(out, None, saved).gate.shape == (0, 1, 50)


def test_norm_rows_that_are_zero_or_not_finite():
    """A zero row normalises to zero with eps; Inf and NaN stay in their rows
    (and in the sums over rows), and their blocks read back NaN."""
    x = rand((6, 100), F32, 1)
    x[1] = 0.0
    x[3, 5], x[4, 70] = math.inf, math.nan
    for norm in ("rms", "layer"):
        y, saved = rf().prenorm(x, None, norm=norm, eps=1e-6)
        assert torch.equal(y[1], torch.zeros(100, device="cuda"))
        assert torch.isfinite(y[[0, 1, 2, 5]]).all() and torch.isnan(y[4]).all() and torch.isnan(y[3, 5])
        g = rf().prenorm_grad(torch.ones_like(x), saved)
        assert torch.isfinite(g.x[[0, 1, 2, 5]]).all() and torch.isnan(g.x[4]).all()


def test_vectors_of_any_stride():
    """Strided weights, biases and gates give the bits of contiguous ones."""
    x, u = rand((30, 100), BF16, 1), rand((30, 100), BF16, 2)
    v = rand((100, 7), F32, 3, 0.2, 1.0)
    gate = rand((100, 3, 30), F32, 4).permute(2, 1, 0)[:, :1]
    args = {"norm": "layer", "next_norm": "layer"}
    r, b = x.view(30, 1, 100), u.view(30, 1, 100)
    first = rf().postnorm_residual(r, b, v[:, 0], v[:, 1], gate, next_weight=v[:, 2], next_bias=v[:, 3], **args)
    c = [v[:, i].contiguous() for i in range(4)]
    second = rf().postnorm_residual(r, b, c[0], c[1], gate.contiguous(), next_weight=c[2], next_bias=c[3], **args)
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    for p, q in zip(rf().postnorm_residual_grad(r, b, first[2]), rf().postnorm_residual_grad(r, b, second[2])):
        assert torch.equal(p, q)


# --------------------------------------------------------- past 32-bit offsets ---
def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: rows near the end are those of a
    call on them alone."""
    rows, cols = 270_000, 8192  # 2.2e9 elements
    last = slice(rows - 40, rows)
    x = torch.empty(rows, cols, dtype=BF16, device="cuda")
    for i in range(0, rows, 27_000):
        x[i: i + 27_000] = rand((1, cols), BF16, i) * torch.linspace(0.5, 2, 27_000, device="cuda").to(BF16)[:, None]
    ck = rf().checkpoint_activations(x)
    end = rf().checkpoint_activations(x[last])
    assert torch.equal(ck.codes[last], end.codes) and torch.equal(ck.exponents[last], end.exponents)
    y = rf().restore_activations(ck)
    assert torch.equal(y[last], rf().restore_activations(end))
    del y
    w = rand((cols,), F32, 1, 0.1, 1.0)
    y, saved = rf().prenorm(x, w)
    y2, saved2 = rf().prenorm(x[last], w)
    assert torch.equal(y[last], y2)
    dx = rf().prenorm_grad(y, saved).x
    assert torch.equal(dx[last], rf().prenorm_grad(y2, saved2).x)
    del y, saved, dx
    h, kept_h = rf().gated_activation(x, x)
    h2, kept_h2 = rf().gated_activation(x[last], x[last])
    assert torch.equal(h[last], h2)
    dg, _ = rf().gated_activation_grad(h, kept_h)
    assert torch.equal(dg[last], rf().gated_activation_grad(h2, kept_h2)[0])
    del h, kept_h, dg, x
    # the sum over all rows, in two calls: f32 sums in another order
    dy = rand((rows, 1), F32, 2).to(BF16).expand(rows, 8).contiguous()
    whole = rf().linear_weight_grad(dy, ck, dtype=F32)
    half = rows // 2
    parts = torch.zeros(8, cols, device="cuda")
    for s in (slice(0, half), slice(half, rows)):
        part = rf().ActivationCheckpoint(ck.codes[s], ck.exponents[s], (ck.codes[s].shape[0], cols), BF16)
        rf().linear_weight_grad(dy[s], part, out=parts, accumulate=True)
    size = (dy[:, :1].float().abs().sum() * 8).item()  # |x| below 8
    assert (whole - parts).abs().max().item() <= 2 * rows ** 0.5 * U * size


@pytest.mark.parametrize("rows,cols,dtype", [(9001, 8195, F32), (18003, 8196, BF16), (36001, 4100, F16)])
def test_restored_outputs_larger_than_the_cache(rows, cols, dtype):
    """Outputs that are stored past the cache, rows that end inside a chunk:
    every run of rows is what restoring it alone gives."""
    x = rand((rows, cols), dtype, 9)
    x *= torch.linspace(0.1, 4, rows, device="cuda").to(dtype)[:, None]
    ck = rf().checkpoint_activations(x)
    y = rf().restore_activations(ck)
    for at in range(0, rows, 1000):
        n = min(1000, rows - at)
        part = rf().ActivationCheckpoint(ck.codes[at: at + n], ck.exponents[at: at + n], (n, cols), dtype)
        assert torch.equal(y[at: at + n], rf().restore_activations(part)), at


# ------------------------------------------------- gradients by differences ---
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_gradients_by_differences(norm):
    """The gradients of a scalar of the f32 operators along random directions,
    against central differences of the 64-bit definition (third derivatives
    of these functions are of order one here: 1e-4 steps leave 1e-7)."""
    rows, cols = 8, 48
    names = ["r", "u", "w", "b", "gate", "w2", "b2"]
    v = {n: rand((rows, cols) if n in "ru" else (cols,), F32, i + 1, 0.3, 1.0 if n[0] in "wg" else 0.0)
         for i, n in enumerate(names)}
    v["u"] = rand((rows, cols), F32, 2, 1.0)
    cout, cy = rand((rows, cols), F32, 20), rand((rows, cols), F32, 21)

    def value(p):
        mean, rstd = stats64(p["u"], norm, 1e-5)
        out = 0.9 * p["r"] + 0.5 * p["gate"] * ((p["u"] - mean) * rstd * p["w"] + p["b"])
        mean, rstd = stats64(out, norm, 1e-5)
        y = (out - mean) * rstd * p["w2"] + p["b2"]
        return (out * d(cout)).sum() + (y * d(cy)).sum()

    _, _, saved = rf().postnorm_residual(v["r"], v["u"], v["w"], v["b"], v["gate"], norm=norm, eps=1e-5,
                                         branch_scale=0.5, residual_scale=0.9, next_norm=norm, next_weight=v["w2"],
                                         next_bias=v["b2"], next_eps=1e-5, save="input")
    grads = dict(zip(names, rf().postnorm_residual_grad(cout, cy, saved)))
    p = {n: d(x) for n, x in v.items()}
    for i, n in enumerate(names):
        way = d(rand(p[n].shape, F32, 30 + i))
        step = 1e-4
        diff = (value({**p, n: p[n] + step * way}) - value({**p, n: p[n] - step * way})) / (2 * step)
        along = (d(grads[n]) * way).sum()
        size = (d(grads[n]) * way).abs().sum()
        assert abs(along - diff) <= 1e-5 * size + 1e-6, (n, along.item(), diff.item())


# ------------------------------------------------------------------ autograd ---
def test_autograd_block_against_torch():
    """A block through the differentiable forms: with save='input' its
    gradients are torch's own (both in f32: 1e-4 of each gradient's norm covers
    the orders of summation); with 8-bit saves they are within 3 % (steps of
    1 / 64 .. 1 / 128 of a block's largest value, independent per element)."""
    ag = rf().autograd
    cols, ffn, rows = 96, 160, 70
    p = {"w": rand((cols,), F32, 1, 0.1, 1.0), "gu": rand((2 * ffn, cols), F32, 2, 0.1), "dn": rand((cols, ffn), F32, 3, 0.1),
         "wo": rand((cols,), F32, 4, 0.1, 1.0), "gate": rand((cols,), F32, 5, 0.1, 0.5), "w2": rand((cols,), F32, 6, 0.1, 1.0)}
    x = rand((5, rows // 5, cols), F32, 7)
    cy, co = rand(x.shape, F32, 8), rand(x.shape, F32, 9)
    for v in (*p.values(), x):
        v.requires_grad_(True)

    def ours(save):
        y, k = ag.prenorm(x, p["w"], save=save, checkpoint_output=True)
        gu = ag.linear(y, p["gu"], checkpoint=k)
        h, k = ag.gated_activation(gu, save=save, checkpoint_output=True)
        br = ag.linear(h, p["dn"], checkpoint=k)
        out, y, _ = ag.postnorm_residual(x, br, p["wo"], gate=p["gate"], next_norm="rms", next_weight=p["w2"], save=save,
                                         checkpoint_output=True)
        return out, y

    def plain():
        n = lambda t, w: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
        gu = n(x, p["w"]) @ p["gu"].t()
        br = (torch.nn.functional.silu(gu[..., :ffn]) * gu[..., ffn:]) @ p["dn"].t()
        out = x + p["gate"] * n(br, p["wo"])
        return out, n(out, p["w2"])

    def grads(f):
        out, y = f()
        return (out, y), torch.autograd.grad((out * co).sum() + (y * cy).sum(), [x, *p.values()])

    (o0, y0), ref = grads(plain)
    for save, bound in (("input", 1e-4), ("int8", 0.03)):
        (o1, y1), got = grads(lambda: ours(save))
        assert torch.allclose(o0, o1, rtol=1e-4, atol=1e-5) and torch.allclose(y0, y1, rtol=1e-4, atol=1e-5)
        for name, a, b in zip(["x", *p], got, ref):
            # the linear layers' inputs are checkpoints in both
            b8 = 0.03 if name in ("gu", "dn") else bound
            assert (a - b).norm() <= b8 * b.norm(), (save, name, ((a - b).norm() / b.norm()).item())
    with torch.no_grad():
        out, y = ours("int8")
        assert torch.equal(out, o1) and not out.requires_grad


def test_autograd_unused_outputs_and_writes():
    ag = rf().autograd
    x, u = rand((9, 40), F32, 1).requires_grad_(True), rand((9, 40), F32, 2).requires_grad_(True)
    out, y = ag.postnorm_residual(x, u, next_norm="rms")
    gx, gu = torch.autograd.grad(out.sum(), [x, u], retain_graph=True)
    assert torch.equal(gx, torch.ones_like(gx)) and torch.isfinite(gu).all()
    gx, gu = torch.autograd.grad(y.square().sum(), [x, u])
    assert torch.isfinite(gx).all() and torch.isfinite(gu).all()
    v = u * 1.0
    h = ag.gated_activation(v, v * 2, save="input")
    with torch.no_grad():
        v.mul_(2)
    with pytest.raises(RuntimeError):
        h.sum().backward()


# --------------------------------------------------------- streams and graphs ---
def test_on_another_stream():
    """Work goes to the current stream, and temporaries are its own."""
    side = torch.cuda.Stream()
    x, u, w = rand((512, 1000), BF16, 1), rand((512, 1000), BF16, 2), rand((1000,), F32, 3)
    torch.cuda.synchronize()

    def step():
        out, y, saved = rf().postnorm_residual(x, u, w, gate=w, next_norm="rms", next_weight=w)
        g = rf().postnorm_residual_grad(x, u, saved)
        dw = rf().linear_weight_grad(g.branch, rf().checkpoint_activations(y), dtype=F32)
        return [out, y, *(t for t in g if t is not None), dw]

    here = step()
    with torch.cuda.stream(side):
        there = step()
    side.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(here, there))


def test_in_a_graph():
    """Captured calls replay with new inputs, between eager work."""
    x, u, w = rand((300, 500), BF16, 1), rand((300, 500), BF16, 2), rand((500,), F32, 3)

    def step():
        out, y, saved = rf().postnorm_residual(x, u, w, gate=w, next_norm="layer", next_weight=w)
        g = rf().postnorm_residual_grad(x, u, saved)
        h, kept_h = rf().gated_activation(y, out)
        dg, du = rf().gated_activation_grad(u, kept_h)
        dw = rf().linear_weight_grad(g.branch, rf().checkpoint_activations(h), dtype=F32)
        return [out, y, *(t for t in g if t is not None), h, dg, du, dw]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        x.copy_(rand((300, 500), BF16, 10 + i))
        u.copy_(rand((300, 500), BF16, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i
