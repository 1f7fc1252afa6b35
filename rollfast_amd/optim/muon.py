"""Orthogonalised updates on MI355X HIP kernels (no reference counterpart here).

``orthogonalize`` brings the singular values of matrices near one by
Newton-Schulz products: with X = G / (|G| + eps), |G| the Frobenius norm, every
step computes

    A = X X^T,  X = a X + (b A + c A^2) X

on the shorter side.  Five steps of the default coefficients bring singular
values from about 0.01 of the norm on to 0.7 .. 1.2, and leave smaller ones
a^5 = 485 times as large.  ``muon8`` is the optimizer made of it: momentum in
8-bit blocks, as ``adamw8`` keeps its moments, orthogonalised.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any, NamedTuple

import numpy as np

from .. import _lib, _tree
from .._base import NO_PARAMS_MSG, GradientTransformationExtraArgs, is_passthrough_leaf, safe_int32_increment
from .adam8 import DYNAMIC_SIGNED_CODEBOOK_ID, QuantizedBlocks, _Config, _init_moment_tree, _rf_dtype, _torch

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_MOST = 256  # matrices of a call of the library


def _steps(steps, coefficients) -> np.ndarray:
    """[steps, 3] f32: the same coefficients in every step, or a row for each."""
    if isinstance(steps, bool) or int(steps) != steps or not 0 <= steps <= 100:
        raise ValueError(f"steps must be a whole number from 0 to 100, got {steps!r}")
    table = np.asarray(coefficients, dtype=np.float32)
    if table.shape == (3,):
        table = np.tile(table, (int(steps), 1))
    if table.shape != (int(steps), 3):
        raise ValueError(f"coefficients must be three numbers, or three for each of the {steps} steps")
    return np.ascontiguousarray(table)


def _matrix_rows(x, what: str):
    """x [rows, cols] with contiguous columns, and its row stride."""
    if x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, (x.stride(0) if x.shape[0] > 1 else x.shape[1])


def orthogonalize(matrices, *, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7, scale: float = 1.0):
    """``scale`` times the orthogonalised matrices of a tree of tensors (or of
    one tensor) [..., rows, cols], in their own dtypes: float32, bfloat16 or
    float16 on one ROCm device.  All of them go through the same launches.

    bfloat16 matrices are worked on in float16 products with what float16 rounds
    away kept beside; float32 and float16 ones in products of split numbers, to
    about 20 bits.  A matrix with an Inf or NaN comes back as NaN; so does a zero
    matrix with ``eps=0``.  ``coefficients``: (a, b, c), or one such row for every
    step; those that let a singular value grow past 64 are refused."""
    torch = _torch()
    table = _steps(steps, coefficients)
    leaves, td = _tree.flatten(matrices)
    out, rows, held, device = [], [], [], None
    for x in leaves:
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"matrices must be torch.Tensors on a ROCm device, got {type(x)}")
        if not x.is_cuda:
            raise ValueError(f"matrices must live on a ROCm device (got {x.device})")
        device = x.device if device is None else device
        if x.device != device:
            raise ValueError("all matrices must live on the same device")
        if x.dim() < 2:
            raise ValueError(f"a matrix has two dimensions at least, got shape {tuple(x.shape)}")
        dtype = _rf_dtype(x.dtype, "matrix")
        y = torch.empty(x.shape, dtype=x.dtype, device=device)
        out.append(y)
        if not x.numel():
            continue
        pairs = [(x, y)] if x.dim() == 2 else list(zip(x.reshape(-1, *x.shape[-2:]), y.view(-1, *x.shape[-2:])))
        for g, o in pairs:
            g, stride = _matrix_rows(g, "matrix")
            held.append(g)
            rows.append(_lib.OrthogonalMatrix(g.data_ptr(), o.data_ptr(), g.shape[0], g.shape[1], stride, o.shape[1], dtype,
                                              scale))
    # results of one precision together
    rows.sort(key=lambda r: r.dtype != _lib.RF_BF16)
    entries = _lib.lib()
    for at in range(0, max(1, len(rows)), _MOST):
        part = rows[at: at + _MOST]
        matrices_ = (_lib.OrthogonalMatrix * len(part))(*part)
        need = ctypes.c_int64()
        _lib.check(entries.rf_orthogonalize_workspace(matrices_, len(part), need), "orthogonalize")
        if device is None:
            continue
        with torch.cuda.device(device):
            workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
            _lib.check(entries.rf_orthogonalize(matrices_, len(part), int(steps), table.ctypes.data, eps,
                                                workspace.data_ptr() or None, need.value, _lib.stream_ptr()),
                       "orthogonalize")
    return _tree.unflatten(td, out)


class Muon8State(NamedTuple):
    """State of ``muon8``: the step count and the momentum, per leaf
    ``QuantizedBlocks`` or, below ``min_size`` elements, a float32 tensor."""

    count: Any
    mu: Any


def _scale_of(shape, adjust: str) -> float:
    rows, cols = shape
    if adjust == "spectral":
        return math.sqrt(max(1.0, rows / cols)) if cols else 1.0
    if adjust == "rms":
        return 0.2 * math.sqrt(max(rows, cols))
    return 1.0


class _Muon8Update:
    """``muon8(...).update``."""

    def __init__(self, learning_rate, momentum, nesterov, weight_decay, steps, table, eps, adjust):
        self.learning_rate, self.momentum, self.nesterov = learning_rate, float(momentum), bool(nesterov)
        self.weight_decay, self.steps, self.table, self.eps, self.adjust = float(weight_decay), steps, table, float(eps), adjust

    def __call__(self, updates, state, params=None, **extra_args):
        del extra_args
        torch = _torch()
        count = int(np.asarray(state.count))
        lr = self.learning_rate
        lr = float(lr(np.asarray(count, dtype=np.int32))) if callable(lr) else float(lr)
        grads, td = _tree.flatten(updates, is_leaf=is_passthrough_leaf)
        moments = _tree.flatten_up_to(td, state.mu)
        if self.weight_decay and params is None:
            raise ValueError(NO_PARAMS_MSG)
        decayed = _tree.flatten_up_to(td, params) if self.weight_decay else [None] * len(grads)
        out, rows, held, device = [], [], [], None
        for g, m, p in zip(grads, moments, decayed):
            if is_passthrough_leaf(g):
                out.append(g)
                continue
            if not isinstance(g, torch.Tensor) or not g.is_cuda:
                raise ValueError("updates must be torch tensors on a ROCm device")
            device = g.device if device is None else device
            _matrix_leaf(g, "updates")
            row = _lib.Muon8Leaf()
            row.dtype, row.block_size = _rf_dtype(g.dtype, "update"), 1
            row.rows, row.cols = g.shape
            if isinstance(m, QuantizedBlocks):
                if m.codebook_id != DYNAMIC_SIGNED_CODEBOOK_ID or m.scales.dtype != torch.float32:
                    raise ValueError("the momentum must be in dynamic signed codes with float32 scales")
                blocks = max(1, -(-m.size // m.block_size))
                if tuple(m.shape) != tuple(g.shape) or m.values.numel() != blocks * m.block_size or m.scales.numel() != blocks:
                    raise ValueError(f"the momentum has shape {tuple(m.shape)}, the gradient {tuple(g.shape)}")
                kept = (m.values, m.scales)
                row.codes, row.scales, row.block_size = m.values.data_ptr(), m.scales.data_ptr(), m.block_size
            else:
                if not isinstance(m, torch.Tensor) or m.shape != g.shape or m.dtype != torch.float32:
                    raise ValueError(f"the momentum must be float32 of shape {tuple(g.shape)}")
                kept = (m,)
                row.momentum = m.data_ptr()
            for t in (*kept, *(() if p is None else (p,))):
                if t.device != device:
                    raise ValueError("all leaves must live on the same device")
            if not all(t.is_contiguous() for t in kept):
                raise ValueError("the momentum must be contiguous")
            if g.device != device:
                raise ValueError("all leaves must live on the same device")
            g = g.contiguous()
            row.grad, row.scale = g.data_ptr(), -lr * _scale_of(g.shape, self.adjust)
            if p is not None:
                if p.shape != g.shape:
                    raise ValueError(f"a parameter has shape {tuple(p.shape)}, its gradient {tuple(g.shape)}")
                p = p.contiguous()
                row.param, row.param_dtype, row.decay = p.data_ptr(), _rf_dtype(p.dtype, "param"), -lr * self.weight_decay
            y = torch.empty(g.shape, dtype=g.dtype, device=device)
            row.update = y.data_ptr()
            out.append(y)
            held += [g, p]
            if g.numel():
                rows.append(row)
        rows.sort(key=lambda r: r.dtype != _lib.RF_BF16)
        entries = _lib.lib()
        for at in range(0, len(rows), _MOST):
            part = rows[at: at + _MOST]
            leaves = (_lib.Muon8Leaf * len(part))(*part)
            need = ctypes.c_int64()
            _lib.check(entries.rf_muon8_update_workspace(leaves, len(part), need), "muon8")
            with torch.cuda.device(device):
                workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
                _lib.check(entries.rf_muon8_update(leaves, len(part), self.momentum, 1.0 - self.momentum, self.nesterov,
                                                   self.steps, self.table.ctypes.data, self.eps, workspace.data_ptr(),
                                                   need.value, _lib.stream_ptr()), "muon8")
        return _tree.unflatten(td, out), Muon8State(np.asarray(safe_int32_increment(count), dtype=np.int32), state.mu)


def _matrix_leaf(x, what: str):
    if x.dim() != 2:
        raise ValueError(f"{what} must be matrices, got shape {tuple(x.shape)}: give other leaves to another "
                         "transformation (multi_transform, masked)")


def muon8(learning_rate, momentum: float = 0.95, *, nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
          coefficients=COEFFICIENTS, eps: float = 1e-7, adjust: str = "spectral", block_size: int = 2048,
          min_size: int = 4096) -> GradientTransformationExtraArgs:
    """Orthogonalised momentum with the momentum in 8-bit blocks:

        m = momentum m + (1 - momentum) g
        u = momentum m + (1 - momentum) g  (nesterov), or m
        update = -lr (s orthogonalize(u) + weight_decay p)

    in the gradient's dtype.  ``adjust`` gives s: 'spectral' sqrt(max(1, rows /
    cols)), 'rms' 0.2 sqrt(max(rows, cols)), None 1.  m is stored as
    ``quantize_blocks`` stores it (dynamic signed codes, one float32 scale per
    ``block_size`` elements), below ``min_size`` elements in float32; u is formed
    from m before that.  A gradient that is not finite makes its matrix' update
    NaN, and leaves the blocks (float32: the elements) that it falls in as they
    were.  Every leaf is a matrix: give embeddings, vectors and the
    like to ``adamw8`` with ``multi_transform``.  ``learning_rate``: a number, or a
    function of the step count.  The momentum is updated in place: the returned
    state shares its tensors."""
    if not 0.0 <= momentum < 1.0:
        raise ValueError(f"momentum must be in [0, 1), got {momentum}")
    if not (math.isfinite(weight_decay) and weight_decay >= 0.0):
        raise ValueError(f"weight_decay must be finite and not negative, got {weight_decay}")
    if block_size <= 0:
        raise ValueError("block_size must be positive.")
    if min_size < 0:
        raise ValueError("min_size must be non-negative.")
    if adjust not in ("spectral", "rms", None):
        raise ValueError(f"adjust must be 'spectral', 'rms' or None, got {adjust!r}")
    table = _steps(steps, coefficients)
    torch = _torch()
    cfg = _Config(0.0, 0.0, 0.0, 0.0, int(block_size), int(min_size), torch.float32, torch.float32, False, "shard_local",
                  True, False, None, False, "jax")

    def init_fn(params):
        for p in _tree.leaves(params, is_leaf=is_passthrough_leaf):
            if not is_passthrough_leaf(p):
                _matrix_leaf(p, "params")
        return Muon8State(np.zeros((), dtype=np.int32), _init_moment_tree(params, cfg, "dynamic_signed"))

    return GradientTransformationExtraArgs(
        init_fn, _Muon8Update(learning_rate, momentum, nesterov, weight_decay, int(steps), table, eps, adjust))
