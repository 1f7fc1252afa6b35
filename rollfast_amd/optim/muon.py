"""Orthogonalised updates on MI355X HIP kernels (no reference counterpart here).

``orthogonalize`` brings the singular values of matrices near one by
Newton-Schulz products: with X = G / (|G| + eps), |G| the Frobenius norm, every
step computes

    A = X X^T,  X = a X + (b A + c A^2) X

on the shorter side.  Five steps of the default coefficients bring singular
values from about 0.01 of the norm on to 0.7 .. 1.2, and leave smaller ones
a^5 = 485 times as large.
"""

from __future__ import annotations

import ctypes

import numpy as np

from .. import _lib, _tree
from .adam8 import _rf_dtype, _torch

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
        pairs = [(x, y)] if x.dim() == 2 else list(zip(x.reshape(-1, *x.shape[-2:]), y.view(-1, *x.shape[-2:])))
        for g, o in pairs:
            if not g.numel():
                continue
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
