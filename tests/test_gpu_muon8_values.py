"""``muon8`` where gradients are not finite, and composed with the other
transformations: clipping, accumulation, the guard, labels."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import oracle as orc
from tests.test_gpu_muon8 import BF16, BOUND, F16, F32, exact, gaussian, low_rank, rf, step

pytestmark = pytest.mark.gpu


def moments(q):
    return [x.clone() for x in ((q.values, q.scales) if isinstance(q, rf().QuantizedBlocks) else (q,))]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("block_size", [16, 100, 512, 2048, 5000])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_gradient_that_is_not_finite_does_not_get_into_the_momentum(value, block_size, dtype):
    """The blocks that it falls in stay as they were, the others are this step's bit for
    bit; the update is NaN, and the next one follows from finite gradients alone."""
    tx = rf().muon8(0.02, block_size=block_size, min_size=0)
    shape, at = (130, 97), [(0, 0), (77, 3), (77, 4), (129, 96)]
    state = tx.init([gaussian(*shape, dtype)])
    _, state = tx.update([low_rank(*shape, dtype, seed=1) * 1e-3], state)
    old = moments(state.mu[0])
    m = rf().dequantize_blocks(state.mu[0]).cpu().numpy()
    bad = low_rank(*shape, dtype, seed=2) * 1e-3
    g = bad.float().cpu().numpy()
    for i, j in at:
        bad[i, j] = value
    updates, state = tx.update([bad], state)
    assert updates[0].isnan().any()
    codes, scales = orc.quantize(step(m, g, 0.95, True)[0], block_size)
    hit = sorted({(i * shape[1] + j) // block_size for i, j in at})
    keep = np.ones(len(scales), bool)
    keep[hit] = False
    got = [x.cpu().numpy().reshape(len(scales), -1) for x in moments(state.mu[0])]
    was = [x.cpu().numpy().reshape(len(scales), -1) for x in old]
    assert np.array_equal(got[0][keep], codes.reshape(len(scales), -1)[keep]) and np.array_equal(got[1][keep, 0], scales[keep])
    assert np.array_equal(got[0][hit], was[0][hit]) and np.array_equal(got[1][hit], was[1][hit])
    now = rf().dequantize_blocks(state.mu[0]).cpu().numpy()
    assert np.isfinite(now).all()
    good = low_rank(*shape, dtype, seed=3) * 1e-3
    updates, state = tx.update([good], state)
    ref = -0.02 * math.sqrt(shape[0] / shape[1]) * exact(torch.from_numpy(step(now, good.float().cpu().numpy(), 0.95, True)[1]).cuda())
    assert (updates[0].double() - ref).norm().item() < BOUND[dtype] * ref.norm().item() * 1.2


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_an_f32_momentum_keeps_the_elements_that_would_not_be_finite(value):
    tx = rf().muon8(0.02, min_size=100000)
    shape = (45, 61)
    state = tx.init([gaussian(*shape, F32)])
    _, state = tx.update([low_rank(*shape, F32, seed=1)], state)
    old = state.mu[0].clone()
    bad = low_rank(*shape, F32, seed=2)
    want = torch.from_numpy(step(old.cpu().numpy(), bad.cpu().numpy(), 0.95, True)[0]).cuda()
    for i, j in ((0, 0), (20, 7), (44, 60)):
        bad[i, j] = value
        want[i, j] = old[i, j]
    updates, state = tx.update([bad], state)
    assert updates[0].isnan().any() and torch.equal(state.mu[0], want)


SPEC = {"embed": (300, 64), "norm": (64,), "up": (256, 64), "down": (64, 256)}
LABELS = {"embed": "rest", "norm": "rest", "up": "matrix", "down": "matrix"}


def tree(seed, dtype=BF16, scale=1e-2):
    return {k: (low_rank(*s, dtype, seed=seed + i) if len(s) == 2 else gaussian(1, *s, dtype, seed=seed)[0]) * scale
            for i, (k, s) in enumerate(SPEC.items())}


def both():
    return rf().multi_transform({"matrix": rf().muon8(0.02, weight_decay=0.1), "rest": rf().adamw8(1e-3)}, LABELS)


def tensors(state):
    """Every tensor of a state, copied."""
    found = []

    def walk(x):
        if isinstance(x, torch.Tensor):
            found.append(x.clone())
        elif isinstance(x, rf().QuantizedBlocks):
            found.extend(moments(x))
        elif isinstance(x, dict):
            for k in sorted(x):
                walk(x[k])
        elif isinstance(x, (list, tuple)):
            for y in x:
                walk(y)

    walk(state)
    return found


def same(a, b):
    assert len(a) == len(b) > 0 and all(torch.equal(x, y) for x, y in zip(a, b))


def same_tree(a, b):
    assert a.keys() == b.keys() and all(torch.equal(a[k], b[k]) for k in a)


MATRICES = ("up", "down")
COMPOSITIONS = {
    "muon8": (lambda: rf().muon8(0.02, weight_decay=0.1), MATRICES),
    "clipped": (lambda: rf().chain(rf().clip_by_global_norm(0.5), rf().muon8(0.02, weight_decay=0.1)), MATRICES),
    "labels": (both, tuple(SPEC)),
    "clipped labels": (lambda: rf().chain(rf().clip_by_global_norm(0.5), both()), tuple(SPEC)),
    "masked": (lambda: rf().masked(rf().muon8(0.02), {"up": True, "down": False}), MATRICES),
    "chained twice": (lambda: rf().chain(rf().clip_by_global_norm(0.5), rf().clip_by_global_norm(0.1), both()), tuple(SPEC)),
}


def part(t, names):
    return {k: t[k] for k in names}


def test_clipped_before_muon8():
    """The chain is the clipping and then the updates."""
    params = part(tree(1), MATRICES)
    tx, alone = COMPOSITIONS["clipped"][0](), rf().muon8(0.02, weight_decay=0.1)
    clip = rf().clip_by_global_norm(0.5)
    state, other, c = tx.init(params), alone.init(params), clip.init(params)
    for turn in range(2):
        grads = part(tree(10 + turn), MATRICES)
        got, state = tx.update(grads, state, params)
        clipped, c = clip.update(grads, c)
        ref, other = alone.update(clipped, other, params)
        same_tree(got, ref)
    same(tensors(state), tensors(other))


@pytest.mark.parametrize("name", COMPOSITIONS)
def test_accumulated(name):
    """MultiSteps of two: the inner update of the mean, zeros before it."""
    make, names = COMPOSITIONS[name]
    params = part(tree(1, F32), names)
    tx, alone = rf().MultiSteps(make(), 2), make()
    state, other = tx.init(params), alone.init(params)
    for turn in range(4):
        grads = part(tree(10 + turn, F32), names)
        got, state = tx.update(grads, state, params)
        if turn % 2 == 0:
            assert not any(x.any() for x in got.values())
            mean = grads
            continue
        # the running mean, each operation rounded
        mean = {k: mean[k] + (grads[k] - mean[k]) * 0.5 for k in names}
        ref, other = alone.update(mean, other, params)
        same_tree(got, ref)
        same(tensors(state.inner_opt_state), tensors(other))


@pytest.mark.parametrize("name", COMPOSITIONS)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_guarded(value, name):
    """apply_if_finite: a step with a value that is not finite anywhere leaves all state
    as it was and gives zeros; accepted steps are the unguarded ones."""
    make, names = COMPOSITIONS[name]
    params = part(tree(1), names)
    tx, alone = rf().apply_if_finite(make(), 2), make()
    state, other = tx.init(params), alone.init(params)
    for turn, bad in enumerate([None, names[0], names[-1], None, None]):
        grads = part(tree(10 + turn), names)
        if bad is not None:
            grads[bad].view(-1)[-1] = value
        before = tensors(state.inner_state)
        got, state = tx.update(grads, state, params)
        assert bool(state.last_finite) == (bad is None)
        if bad is not None:
            assert all(x.dtype == grads[k].dtype and not x.any() for k, x in got.items())
            same(before, tensors(state.inner_state))
            continue
        ref, other = alone.update(grads, other, params)
        same_tree(got, ref)
        same(tensors(state.inner_state), tensors(other))
    assert int(state.total_notfinite) == 2 and int(state.notfinite_count) == 0
    # more in a row than are allowed: the third goes through
    for turn in range(3):
        grads = part(tree(30 + turn), names)
        grads["up"][0, 0] = value
        got, state = tx.update(grads, state, params)
        assert int(state.notfinite_count) == turn + 1
        assert got["up"].isfinite().all() == (turn < 2)


def test_guarded_inside_an_accumulation():
    """As the builders of a fine-tuning step nest them."""
    params = tree(1, F32)
    tx = rf().MultiSteps(rf().apply_if_finite(rf().chain(rf().clip_by_global_norm(0.5), both()), 1), 2)
    state = tx.init(params)
    before = tensors(state.inner_opt_state)
    for turn in range(2):
        grads = tree(10 + turn, F32)
        grads["norm"][3] = math.nan
        got, state = tx.update(grads, state, params)
        assert not any(x.any() for x in got.values())
    same(before, tensors(state.inner_opt_state))
    assert int(state.inner_opt_state.total_notfinite) == 1
    # (the accumulator's reset is a product with zero, which leaves a NaN one: begun again)
    alone, state = rf().chain(rf().clip_by_global_norm(0.5), both()), tx.init(params)
    grads = tree(20, F32)
    for _ in range(2):
        got, state = tx.update(grads, state, params)
    same_tree(got, alone.update(grads, alone.init(params), params)[0])


def test_leaves_of_every_kind_are_tested():
    """Empty ones, strided ones, every dtype, none, the last element of a large one."""
    from rollfast_amd.transforms import _all_finite

    x = gaussian(1000, 999, F32)
    for t in ([], [None], [x[:0]], [x], [x.t(), None, x.to(BF16), x[:, 3:7].to(F16)], [x[3:], x[:0], x]):
        assert _all_finite(t)
    x[999, 998] = math.inf
    assert not _all_finite([x.clone().zero_(), x]) and not _all_finite([x.t()]) and _all_finite([x[:, :998]])
    assert not _all_finite([x.to(BF16)]) and not _all_finite([x.to(F16)])
    big = torch.full((3,), 3e38, device="cuda")
    assert _all_finite([big, big])


def test_fused_steps_refuse_muon8():
    params = tree(1)
    for tx in (rf().apply_if_finite(both(), 1), both(), rf().MultiSteps(both(), 2), rf().muon8(0.1)):
        p = params if tx.update.__class__.__name__ != "_Muon8Update" else part(params, MATRICES)
        with pytest.raises((NotImplementedError, TypeError)):
            state = tx.init(p)
            for _ in range(2):
                _, state = rf().adamw8_step(tx, p, {k: x.clone() for k, x in p.items()}, state, stochastic=False)
