"""``muon8`` against its definition: the stored momentum bit for bit (f32 operations
in order, the CPU oracle's codes), the updates in 64 bits from the momentum as
computed, within the orthogonalisation's bounds (tests/test_gpu_orthogonalize.py)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import oracle as orc
from tests.test_gpu_orthogonalize import BF16, BOUND, F16, F32, exact, gaussian, low_rank

pytestmark = pytest.mark.gpu


def rf():
    import rollfast_amd

    return rollfast_amd


def step(m, g, beta, nesterov):
    """(m, u) in f32, each operation rounded."""
    beta, rest = np.float32(beta), np.float32(1.0 - beta)
    m = beta * m + rest * g
    return m, (beta * m + rest * g if nesterov else m)


SHAPES = [(64, 64), (1, 5), (65, 130), (257, 31), (300, 768), (129, 1025)]


@pytest.mark.parametrize("dtype", [BF16, F32, F16])
@pytest.mark.parametrize("block_size", [2048, 256, 100, 5000])
@pytest.mark.parametrize("nesterov", [True, False])
def test_steps(nesterov, block_size, dtype):
    lr, beta, wd = 0.02, 0.95, 0.1
    tx = rf().muon8(lr, beta, nesterov=nesterov, weight_decay=wd, block_size=block_size, min_size=1000)
    params = {str(i): gaussian(r, c, dtype, seed=i) for i, (r, c) in enumerate(SHAPES)}
    state = tx.init(params)
    host = {k: np.zeros(p.shape, np.float32) for k, p in params.items()}
    for turn in range(3):
        grads = {k: low_rank(*p.shape, dtype, seed=10 * turn + int(k), noise=0.3) * 1e-3 for k, p in params.items()}
        updates, state = tx.update(grads, state, params)
        assert int(state.count) == turn + 1
        for k, p in params.items():
            m, u = step(host[k], grads[k].float().cpu().numpy(), beta, nesterov)
            if p.numel() >= 1000:
                codes, scales = orc.quantize(m, block_size)
                kept = state.mu[k]
                assert np.array_equal(kept.values.cpu().numpy(), codes), (k, turn)
                assert np.array_equal(kept.scales.cpu().numpy().view(np.uint32), scales.view(np.uint32))
                host[k] = orc.dequantize(codes, scales, m.size, block_size).reshape(m.shape)
            else:
                assert np.array_equal(state.mu[k].cpu().numpy(), m)
                host[k] = m
            r, c = p.shape
            ref = -lr * (math.sqrt(max(1.0, r / c)) * exact(torch.from_numpy(u).cuda()) + wd * p.double())
            assert updates[k].dtype == dtype
            # sums of two terms may cancel: the bound is of the terms' norms
            size = lr * (math.sqrt(max(1.0, r / c)) * math.sqrt(min(r, c)) * 1.2 + wd * p.double().norm().item())
            assert (updates[k].double() - ref).norm().item() < BOUND[dtype] * size, (k, turn)


def test_adjust_schedule_and_passthrough():
    g = low_rank(40, 90, F32)
    for adjust, s in (("spectral", 1.0), ("rms", 0.2 * math.sqrt(90)), (None, 1.0)):
        tx = rf().muon8(lambda count: 0.5 / (1 + int(count)), adjust=adjust, min_size=0)
        state = tx.init({"a": g, "b": None, "c": rf().MaskedNode()})
        for turn in range(2):
            old = rf().dequantize_blocks(state.mu["a"]).cpu().numpy()
            updates, state = tx.update({"a": g, "b": None, "c": rf().MaskedNode()}, state)
            assert updates["b"] is None and updates["c"] == rf().MaskedNode()
            u = torch.from_numpy(step(old, g.cpu().numpy(), 0.95, True)[1]).cuda()
            ref = -0.5 / (1 + turn) * s * exact(u)
            assert ((updates["a"].double() - ref).norm() / ref.norm()).item() < BOUND[F32], (adjust, turn)


def test_layouts_and_shared_memory():
    p = gaussian(70, 140, BF16, seed=1)
    g = low_rank(70, 140, BF16, seed=2)
    tx = rf().muon8(0.1, weight_decay=0.01, min_size=0, block_size=256)
    ref, state = tx.update([g], tx.init([p]), [p])
    wide = torch.empty(70, 150, dtype=BF16, device="cuda")
    wide[:, 3:143] = g
    got, other = tx.update([wide[:, 3:143]], tx.init([p]), [p.t().contiguous().t()])
    assert torch.equal(got[0], ref[0]) and torch.equal(other.mu[0].values, state.mu[0].values)
    # the state is updated in place
    before = state.mu[0].values.data_ptr()
    _, state = tx.update([g], state, [p])
    assert state.mu[0].values.data_ptr() == before


def test_empty_matrices_and_none():
    p = {"a": torch.zeros(0, 4, device="cuda"), "b": None}
    tx = rf().muon8(0.1)
    updates, _ = tx.update(p, tx.init(p))
    assert updates["a"].shape == (0, 4) and updates["b"] is None


def test_a_gradient_that_is_not_finite_stays_in_its_matrix():
    grads = [low_rank(80, 64, F32, seed=i) for i in range(3)]
    tx = rf().muon8(0.1, min_size=0)
    ref, _ = tx.update(grads, tx.init(grads))
    bad = [g.clone() for g in grads]
    bad[1][5, 5] = math.nan
    got, _ = tx.update(bad, tx.init(bad))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[2], ref[2]) and got[1].isnan().all()


def test_captured_and_replayed():
    """The momentum goes on from replay to replay as it does from call to call."""
    g, p = low_rank(130, 200, BF16, seed=1), gaussian(130, 200, BF16, seed=2)
    tx = rf().muon8(0.1, weight_decay=0.1)
    eager = tx.init([p])
    tx.update([g], tx.init([p]), [p])
    state = tx.init([p])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = tx.update([g], state, [p])
    state.mu[0].values.copy_(eager.mu[0].values)
    state.mu[0].scales.copy_(eager.mu[0].scales)
    for turn in range(4):
        g.copy_(low_rank(130, 200, BF16, seed=20 + turn))
        graph.replay()
        torch.cuda.synchronize()
        ref, eager = tx.update([g], eager, [p])
        assert torch.equal(got[0], ref[0]) and torch.equal(state.mu[0].values, eager.mu[0].values), turn


def test_with_adamw8_for_the_other_leaves():
    """Matrices to muon8, vectors and the embedding to adamw8, in one transformation."""
    params = {"embed": gaussian(500, 64, BF16, seed=1), "norm": torch.ones(64, dtype=BF16, device="cuda"),
              "up": gaussian(256, 64, BF16, seed=2), "down": gaussian(64, 256, BF16, seed=3)}
    labels = {"embed": "rest", "norm": "rest", "up": "matrix", "down": "matrix"}
    tx = rf().multi_transform({"matrix": rf().muon8(0.02, weight_decay=0.1), "rest": rf().adamw8(1e-3)}, labels)
    state = tx.init(params)
    single = rf().muon8(0.02, weight_decay=0.1)
    alone = single.init({k: params[k] for k in ("up", "down")})
    adam = rf().adamw8(1e-3)
    rest = adam.init({k: params[k] for k in ("embed", "norm")})
    for turn in range(3):
        grads = {k: (low_rank(*p.shape, BF16, seed=turn) if p.dim() == 2 else gaussian(1, 64, BF16, seed=turn)[0]) for k, p in params.items()}
        updates, state = tx.update(grads, state, params)
        a, alone = single.update({k: grads[k] for k in alone.mu}, alone, {k: params[k] for k in alone.mu})
        b, rest = adam.update({k: grads[k] for k in ("embed", "norm")}, rest, {k: params[k] for k in ("embed", "norm")})
        for k in params:
            assert torch.equal(updates[k], (a if k in a else b)[k]), (k, turn)
        params = rf().apply_updates(params, updates, stochastic=False) if turn == 0 else params


@pytest.mark.parametrize("block_size", [1, 4, 8, 16, 64, 512, 1024, 4096])
@pytest.mark.parametrize("count", [1, 5])
def test_block_sizes(count, block_size):
    """Blocks that a wave takes several of, and others; in one list or many."""
    tx = rf().muon8(0.02, block_size=block_size, min_size=0)
    params = [gaussian(r, c, F32, seed=i) for i, (r, c) in enumerate([(257, 31), (1, 5), (64, 64), (130, 515), (9, 57)][:count])]
    state = tx.init(params)
    host = [np.zeros(p.shape, np.float32) for p in params]
    for turn in range(2):
        grads = [low_rank(*p.shape, F32, seed=10 * turn + i, noise=0.3) for i, p in enumerate(params)]
        grads[0][3] = 0.0  # a row of nothing: blocks with a scale of their own
        updates, state = tx.update(grads, state, params)
        for i, p in enumerate(params):
            m, u = step(host[i], grads[i].cpu().numpy(), 0.95, True)
            codes, scales = orc.quantize(m, block_size)
            assert np.array_equal(state.mu[i].values.cpu().numpy(), codes), (i, turn)
            assert np.array_equal(state.mu[i].scales.cpu().numpy().view(np.uint32), scales.view(np.uint32)), (i, turn)
            host[i] = orc.dequantize(codes, scales, m.size, block_size).reshape(m.shape)
            r, c = p.shape
            ref = -0.02 * math.sqrt(max(1.0, r / c)) * exact(torch.from_numpy(u).cuda())
            assert (updates[i].double() - ref).norm().item() < BOUND[F32] * ref.norm().item() * 1.2, (i, turn)
