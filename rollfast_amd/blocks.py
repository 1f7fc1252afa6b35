"""Residual-block operators with 8-bit saved activations (no reference counterpart).

``adamw8`` keeps the optimizer state in 8-bit blocks; what then fills a
training GPU are the activations that the backward pass needs.  These
operators keep them in 8-bit blocks too, and read them from there:

- ``checkpoint_activations`` / ``restore_activations``: an activation into
  8 bits and back;
- ``linear_weight_grad``: a linear layer's weight gradient from its input's
  checkpoint;
- ``gated_activation``: ``act(gate) * up``;
- ``prenorm``: the norm before a block;
- ``postnorm_residual``: the norm after it with its gate, the residual sum
  and, in the same pass, the norm before the next block.

Each forward function returns its outputs and what its ``*_grad`` function
needs (``save="int8"``: 8-bit checkpoints; ``save="input"``: the tensors
themselves, which must then not be written before the backward pass;
``save=None``: nothing, for inference).  ``rollfast_amd.autograd`` has them as
differentiable functions.

A checkpoint has int8 codes and one power-of-two step for every 32 columns of
a row: 1.03 bytes an element.  With E the exponent of a block's largest
magnitude the step is 2^(E - 6), the error at most half a step, or a step
where the magnitude rounds past 127 steps.  A block with an Inf or NaN reads
back as NaN.

Tensors are float32, bfloat16 or float16 on a ROCm device, rows along the last
dimension; any row stride is read in place.  Work is enqueued on the current
stream.  Sums are f32 in a fixed order: equal inputs give equal bits.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any, NamedTuple, Optional

import torch

from . import _lib

BLOCK = 32  # columns that share a step

_DTYPE = {torch.float32: _lib.RF_F32, torch.bfloat16: _lib.RF_BF16, torch.float16: _lib.RF_F16}
_NORM = {"rms": _lib.RF_NORM_RMS, "layer": _lib.RF_NORM_LAYER}
_POST = {"none": _lib.RF_NORM_NONE, **_NORM}
_ACT = {"silu": _lib.RF_ACT_SILU, "gelu": _lib.RF_ACT_GELU, "gelu_tanh": _lib.RF_ACT_GELU_TANH}
_SAVE = ("int8", "input", None)


class ActivationCheckpoint(NamedTuple):
    """An activation in 8-bit blocks: ``codes`` int8 [rows, pitch] (pitch: the
    columns rounded up to 32), ``exponents`` uint8 [rows, pitch // 32] (the
    step's biased exponent), and the shape and dtype of what it stands for."""

    codes: Any
    exponents: Any
    shape: tuple
    dtype: Any

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()


class PrenormGrads(NamedTuple):
    x: Any
    weight: Any
    bias: Any


class PostnormGrads(NamedTuple):
    residual: Any
    branch: Any
    weight: Any
    bias: Any
    gate: Any
    next_weight: Any
    next_bias: Any


class NormSaved:
    """What ``prenorm_grad`` / ``postnorm_residual_grad`` need.  ``output``:
    the checkpoint of y, if one was asked for."""

    __slots__ = ("args", "shape", "dtype", "branch_dtype", "branch", "branch_exponents", "hidden", "hidden_exponents",
                 "post_mean", "post_rstd", "next_mean", "next_rstd", "weight", "bias", "gate", "next_weight",
                 "next_bias", "output")


class GatedSaved:
    """What ``gated_activation_grad`` needs.  ``output``: the checkpoint of h,
    if one was asked for."""

    __slots__ = ("activation", "shape", "dtype", "fused", "gate", "gate_exponents", "up", "up_exponents", "output")


# --------------------------------------------------------------- arguments ---
def _code(dtype, what: str) -> int:
    code = _DTYPE.get(dtype)
    if code is None:
        raise NotImplementedError(f"{what} dtype {dtype} is not supported (float32, bfloat16 or float16)")
    return code


def _tensor(x, what: str, device=None):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor on a ROCm device, got {type(x)}")
    if not x.is_cuda:
        raise ValueError(f"{what} must live on a ROCm device (got {x.device})")
    if device is not None and x.device != device:
        raise ValueError(f"{what} is on {x.device}, expected {device}")
    return x


def _rows(x, what: str):
    """x as (a tensor of rows with contiguous columns, row stride)."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what} needs a last dimension of at least one column")
    cols = x.shape[-1]
    if x.is_contiguous():
        return x, cols
    x = x.reshape(x.numel() // cols, cols)
    if cols > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, x.stride(0)


def _like(x, shape, dtype, what: str, device):
    """Rows of a tensor that must have this shape and dtype."""
    _tensor(x, what, device)
    if x.shape != shape:
        raise ValueError(f"{what} has shape {tuple(x.shape)}, expected {tuple(shape)}")
    if x.dtype != dtype:
        raise ValueError(f"{what} is {x.dtype}, expected {dtype}")
    return _rows(x, what)


def _vector(x, cols: int, what: str, device):
    if x is None:
        return None
    _tensor(x, what, device)
    if x.shape != (cols,):
        raise ValueError(f"{what} has shape {tuple(x.shape)}, expected {(cols,)}")
    _code(x.dtype, what)
    return x.contiguous()


def _gates(gate, shape, device):
    """(the gate's rows, their number): [cols], or shaped like the rows with
    ones after the leading dimensions that it varies over."""
    if gate is None:
        return None, 0
    _tensor(gate, "gate", device)
    _code(gate.dtype, "gate")
    lead, own = tuple(shape[:-1]), tuple(gate.shape[:-1])
    vary = 0
    while vary < len(own) and own[vary:] != (1,) * (len(own) - vary):
        vary += 1
    if not gate.dim() or gate.shape[-1] != shape[-1] or (own and (len(own) != len(lead) or own[:vary] != lead[:vary])):
        raise ValueError(
            f"gate has shape {tuple(gate.shape)}: expected {(shape[-1],)}, or {tuple(shape)} with ones in place of the "
            "dimensions just before the last that share a gate"
        )
    gates = math.prod(own[:vary])
    return (gate.contiguous() if gates else gate), gates  # no gates: no rows


def _check_save(save, checkpoint_output: bool):
    if save not in _SAVE:
        raise ValueError(f"save must be 'int8', 'input' or None, got {save!r}")
    if checkpoint_output and save is None:
        raise ValueError("checkpoint_output needs save='int8' or 'input'")


def _norm_code(norm, table, what: str) -> int:
    if norm not in table:
        raise ValueError(f"{what} must be one of {', '.join(map(repr, table))}, got {norm!r}")
    return table[norm]


def _new_codes(rows: int, cols: int, device):
    blocks = -(-cols // BLOCK)
    return (torch.empty((rows, blocks * BLOCK), dtype=torch.int8, device=device),
            torch.empty((rows, blocks), dtype=torch.uint8, device=device))


def _check_checkpoint(kept, device=None):
    codes, exps = _tensor(kept.codes, "codes", device), _tensor(kept.exponents, "exponents", kept.codes.device)
    shape = tuple(kept.shape)
    if not shape or shape[-1] < 1:
        raise ValueError("a checkpoint's shape needs a last dimension of at least one column")
    rows, blocks = math.prod(shape[:-1]), -(-shape[-1] // BLOCK)
    if codes.dtype != torch.int8 or exps.dtype != torch.uint8:
        raise ValueError("a checkpoint has int8 codes and uint8 exponents")
    if codes.numel() != rows * blocks * BLOCK or exps.numel() != rows * blocks:
        raise ValueError(f"a checkpoint of shape {shape} has codes {(rows, blocks * BLOCK)} and exponents {(rows, blocks)}")
    if not codes.is_contiguous() or not exps.is_contiguous():
        raise ValueError("a checkpoint's codes and exponents must be contiguous")
    return rows, shape[-1]


# -------------------------------------------------------------- checkpoints ---
def checkpoint_activations(x) -> ActivationCheckpoint:
    """x in 8-bit blocks of 32 columns."""
    _tensor(x, "x")
    code = _code(x.dtype, "x")
    v, stride = _rows(x, "x")
    cols = x.shape[-1]
    rows = x.numel() // cols
    codes, exps = _new_codes(rows, cols, x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().rf_checkpoint_store(v.data_ptr(), code, rows, cols, stride, codes.data_ptr(),
                                                  exps.data_ptr(), _lib.stream_ptr()), "checkpoint_activations")
    return ActivationCheckpoint(codes, exps, tuple(x.shape), x.dtype)


def restore_activations(checkpoint: ActivationCheckpoint, *, dtype=None):
    """The values of a checkpoint, in its own dtype or another."""
    dtype = checkpoint.dtype if dtype is None else dtype
    code = _code(dtype, "output")
    rows, cols = _check_checkpoint(checkpoint)
    out = torch.empty(checkpoint.shape, dtype=dtype, device=checkpoint.codes.device)
    with torch.cuda.device(out.device):
        _lib.check(_lib.lib().rf_checkpoint_load(checkpoint.codes.data_ptr(), checkpoint.exponents.data_ptr(), rows, cols,
                                                 code, out.data_ptr(), _lib.stream_ptr()), "restore_activations")
    return out


def linear_weight_grad(dy, checkpoint: ActivationCheckpoint, *, out=None, accumulate: bool = False, dtype=None):
    """The gradient of ``weight`` [outs, cols] in ``y = x @ weight.T`` from
    ``dy`` [..., outs] and the checkpoint of x [..., cols].  ``out``: written,
    or added to with ``accumulate``; else a new tensor of ``dtype`` (dy's)."""
    _tensor(dy, "dy")
    rows, cols = _check_checkpoint(checkpoint, dy.device)
    if dy.dim() == 0 or dy.shape[:-1] != tuple(checkpoint.shape[:-1]):
        raise ValueError(f"dy has shape {tuple(dy.shape)}, the checkpoint {tuple(checkpoint.shape)}: their rows differ")
    v, stride = _rows(dy, "dy")
    outs = dy.shape[-1]
    if stride >= 1 << 24:  # the kernel addresses a few rows by 32 bits
        v, stride = v.contiguous(), outs
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = torch.empty((outs, cols), dtype=dy.dtype if dtype is None else dtype, device=dy.device)
    else:
        _tensor(out, "out", dy.device)
        if out.shape != (outs, cols) or not out.is_contiguous():
            raise ValueError(f"out must be contiguous with shape {(outs, cols)}, got {tuple(out.shape)}")
        if dtype is not None and dtype != out.dtype:
            raise ValueError(f"out is {out.dtype}, dtype says {dtype}")
    a = _lib.WeightGrad()
    a.rows, a.outs, a.cols = rows, outs, cols
    a.dy_dtype, a.out_dtype = _code(dy.dtype, "dy"), _code(out.dtype, "out")
    a.dy, a.dy_stride = v.data_ptr(), stride
    a.codes, a.exponents = checkpoint.codes.data_ptr(), checkpoint.exponents.data_ptr()
    a.out, a.accumulate = out.data_ptr(), int(accumulate)
    with torch.cuda.device(dy.device):
        space, size = _workspace(_lib.lib().rf_linear_weight_grad_workspace, a, dy.device, "linear_weight_grad")
        _lib.check(_lib.lib().rf_linear_weight_grad(a, space, size, _lib.stream_ptr()), "linear_weight_grad")
    return out


def _workspace(query, args, device, what: str):
    """(device pointer, bytes) of a call's workspace: memory of the current
    stream, which torch hands out again only behind the call's work."""
    size = ctypes.c_int64()
    _lib.check(query(args, size), what)
    if not size.value:
        return None, 0
    return torch.empty(size.value, dtype=torch.uint8, device=device).data_ptr(), size.value


# ---------------------------------------------------------- gated activation ---
def gated_activation(gate, up=None, *, activation: str = "silu", save: Optional[str] = "int8",
                     checkpoint_output: bool = False):
    """``h = act(gate) * up`` -> (h, saved).  Without ``up`` the gate's last
    dimension holds both, the gate first (one product's output).
    ``activation``: 'silu', 'gelu' (with the error function) or 'gelu_tanh'."""
    _check_save(save, checkpoint_output)
    if activation not in _ACT:
        raise ValueError(f"activation must be one of {', '.join(map(repr, _ACT))}, got {activation!r}")
    _tensor(gate, "gate")
    code = _code(gate.dtype, "gate")
    fused = up is None
    if fused:
        if gate.dim() == 0 or gate.shape[-1] == 0 or gate.shape[-1] % 2:
            raise ValueError(f"without up the gate's last dimension holds both halves, got shape {tuple(gate.shape)}")
        both, stride = _rows(gate, "gate")
        cols = gate.shape[-1] // 2
        both = both.as_strided((gate.numel() // (2 * cols), 2 * cols), (stride, 1))
        g, u, gs, us = both[:, :cols], both[:, cols:], stride, stride
    else:
        g, gs = _rows(gate, "gate")
        u, us = _like(up, gate.shape, gate.dtype, "up", gate.device)
        cols = gate.shape[-1]
    shape = (*gate.shape[:-1], cols)
    rows, device = math.prod(shape[:-1]), gate.device
    h = torch.empty(shape, dtype=gate.dtype, device=device)
    a = _lib.Gated()
    a.rows, a.cols, a.dtype, a.activation = rows, cols, code, _ACT[activation]
    a.gate, a.up, a.gate_stride, a.up_stride, a.h = g.data_ptr(), u.data_ptr(), gs, us, h.data_ptr()
    saved = None
    if save is not None:
        saved = GatedSaved()
        saved.activation, saved.shape, saved.dtype, saved.fused = activation, shape, gate.dtype, fused
        saved.output = saved.gate_exponents = saved.up_exponents = None
        if save == "int8":
            (saved.gate, saved.gate_exponents), (saved.up, saved.up_exponents) = (_new_codes(rows, cols, device)
                                                                                  for _ in range(2))
            a.gate_codes, a.gate_exponents = saved.gate.data_ptr(), saved.gate_exponents.data_ptr()
            a.up_codes, a.up_exponents = saved.up.data_ptr(), saved.up_exponents.data_ptr()
        else:
            saved.gate, saved.up = g.as_strided((rows, cols), (gs, 1)), u.as_strided((rows, cols), (us, 1))
        if checkpoint_output:
            saved.output = ActivationCheckpoint(*_new_codes(rows, cols, device), shape, gate.dtype)
            a.h_codes, a.h_exponents = saved.output.codes.data_ptr(), saved.output.exponents.data_ptr()
    with torch.cuda.device(device):
        _lib.check(_lib.lib().rf_gated_forward(a, _lib.stream_ptr()), "gated_activation")
    return h, saved


def gated_activation_grad(dh, saved: GatedSaved):
    """(dgate, dup); one tensor that holds both where the forward pass took one."""
    shape, dtype, device = saved.shape, saved.dtype, saved.gate.device
    v, stride = _like(dh, shape, dtype, "dh", device)
    cols = shape[-1]
    rows = math.prod(shape[:-1])
    a = _lib.Gated()
    a.rows, a.cols, a.dtype, a.activation = rows, cols, _DTYPE[dtype], _ACT[saved.activation]
    if saved.gate_exponents is not None:
        a.gate_codes, a.gate_exponents = saved.gate.data_ptr(), saved.gate_exponents.data_ptr()
        a.up_codes, a.up_exponents = saved.up.data_ptr(), saved.up_exponents.data_ptr()
    else:
        a.gate, a.gate_stride = saved.gate.data_ptr(), saved.gate.stride(0)
        a.up, a.up_stride = saved.up.data_ptr(), saved.up.stride(0)
    a.dh, a.dh_stride = v.data_ptr(), stride
    if saved.fused:
        out = torch.empty((*shape[:-1], 2 * cols), dtype=dtype, device=device)
        a.dgate, a.dup = out.data_ptr(), out.data_ptr() + cols * out.element_size()
        a.dgate_stride = a.dup_stride = 2 * cols
    else:
        out = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
        a.dgate, a.dup = out[0].data_ptr(), out[1].data_ptr()
        a.dgate_stride = a.dup_stride = cols
    with torch.cuda.device(device):
        _lib.check(_lib.lib().rf_gated_backward(a, _lib.stream_ptr()), "gated_activation_grad")
    return out


# ---------------------------------------------------------------------- norms ---
def _put_vector(a, name: str, v):
    if v is not None:
        setattr(a, name, v.data_ptr())
        setattr(a, name + "_dtype", _DTYPE[v.dtype])


def _stats(a, part: str, kind: int, rows: int, device, saved):
    """The row statistics that the backward pass needs, one buffer a part."""
    mean = kind == _lib.RF_NORM_LAYER
    if kind not in (_lib.RF_NORM_RMS, _lib.RF_NORM_LAYER):
        return
    rstd = torch.empty(rows * (2 if mean else 1), dtype=torch.float32, device=device)
    setattr(a, part + "_rstd", rstd.data_ptr())
    setattr(saved, part + "_rstd", rstd)
    if mean:
        setattr(a, part + "_mean", rstd.data_ptr() + 4 * rows)


def _new_saved():
    saved = NormSaved()
    for name in NormSaved.__slots__:
        setattr(saved, name, None)
    return saved


def prenorm(x, weight=None, bias=None, *, norm: str = "rms", eps: float = 1e-6, dtype=None,
            save: Optional[str] = "int8", checkpoint_output: bool = False):
    """The norm before a block -> (y, saved):
    ``y = (x - mean) / sqrt(mean((x - mean)^2) + eps) * weight + bias`` for
    norm='layer', without the means for 'rms'.  ``dtype``: y's (x's; a 16-bit
    type beside a float32 x)."""
    _check_save(save, checkpoint_output)
    _tensor(x, "x")
    device, cols = x.device, x.shape[-1] if x.dim() else 0
    v, stride = _rows(x, "x")
    rows = x.numel() // cols
    a = _lib.Norm()
    a.rows, a.cols = rows, cols
    a.dtype, a.next, a.next_eps = _code(x.dtype, "x"), _norm_code(norm, _NORM, "norm"), eps
    out_dtype = x.dtype if dtype is None else dtype
    a.branch_dtype = _code(out_dtype, "y")
    weight, bias = _vector(weight, cols, "weight", device), _vector(bias, cols, "bias", device)
    _put_vector(a, "next_weight", weight)
    _put_vector(a, "next_bias", bias)
    y = torch.empty(x.shape, dtype=out_dtype, device=device)
    a.hidden, a.hidden_stride, a.y = v.data_ptr(), stride, y.data_ptr()
    saved = None
    if save is not None:
        saved = _new_saved()
        saved.shape, saved.dtype, saved.branch_dtype = x.shape, x.dtype, out_dtype
        saved.next_weight, saved.next_bias = weight, bias
        _stats(a, "next", a.next, rows, device, saved)
        _keep(a, "hidden", save, v, stride, rows, cols, device, saved)
        _keep_output(a, checkpoint_output, rows, cols, x.shape, out_dtype, device, saved)
        saved.args = (rows, cols, 0, _lib.RF_NORM_ABSENT, a.next, 1.0, 1.0)
    with torch.cuda.device(device):
        _lib.check(_lib.lib().rf_norm_forward(a, _lib.stream_ptr()), "prenorm")
    return y, saved


def _keep(a, name: str, save: str, v, stride: int, rows: int, cols: int, device, saved):
    if save == "int8":
        codes, exps = _new_codes(rows, cols, device)
        setattr(a, name + "_codes", codes.data_ptr())
        setattr(a, name + "_exponents", exps.data_ptr())
        setattr(saved, name, codes)
        setattr(saved, name + "_exponents", exps)
    else:
        setattr(saved, name, v.as_strided((rows, cols), (stride, 1)))


def _keep_output(a, wanted: bool, rows: int, cols: int, shape, dtype, device, saved):
    if wanted:
        saved.output = ActivationCheckpoint(*_new_codes(rows, cols, device), tuple(shape), dtype)
        a.y_codes, a.y_exponents = saved.output.codes.data_ptr(), saved.output.exponents.data_ptr()


def postnorm_residual(residual, branch, weight=None, bias=None, gate=None, *, norm: str = "rms", eps: float = 1e-6,
                      branch_scale: float = 1.0, residual_scale: float = 1.0, next_norm: Optional[str] = None,
                      next_weight=None, next_bias=None, next_eps: float = 1e-6, save: Optional[str] = "int8",
                      checkpoint_output: bool = False):
    """The end of a block -> (out, y, saved):
    ``out = residual_scale * residual + branch_scale * gate * norm(branch)``
    and, with ``next_norm``, ``y = next_norm(out)``, the input of the next
    block (else None).  ``norm='none'`` leaves the branch as it is.  ``gate``:
    [cols], or the residual's shape with ones for the dimensions before the
    last that share a gate ([sequences, 1, cols] for a gate per sequence).
    ``branch`` and y have one dtype: the residual's, or 16 bits beside a
    float32 residual."""
    _check_save(save, checkpoint_output)
    if checkpoint_output and next_norm is None:
        raise ValueError("checkpoint_output needs next_norm")
    _tensor(residual, "residual")
    _tensor(branch, "branch", residual.device)
    device, cols = residual.device, residual.shape[-1] if residual.dim() else 0
    r, rs = _rows(residual, "residual")
    u, us = _like(branch, residual.shape, branch.dtype, "branch", device)
    rows = residual.numel() // cols
    a = _lib.Norm()
    a.rows, a.cols = rows, cols
    a.dtype, a.branch_dtype = _code(residual.dtype, "residual"), _code(branch.dtype, "branch")
    a.post, a.post_eps = _norm_code(norm, _POST, "norm"), eps
    if a.post == _lib.RF_NORM_NONE and (weight is not None or bias is not None):
        raise ValueError("norm='none' takes no weight or bias")
    a.branch_scale, a.residual_scale = branch_scale, residual_scale
    weight, bias = _vector(weight, cols, "weight", device), _vector(bias, cols, "bias", device)
    gate_rows, a.gates = _gates(gate, residual.shape, device)
    _put_vector(a, "weight", weight)
    _put_vector(a, "bias", bias)
    _put_vector(a, "gate", gate_rows)
    out = torch.empty(residual.shape, dtype=residual.dtype, device=device)
    a.residual, a.residual_stride, a.branch, a.branch_stride = r.data_ptr(), rs, u.data_ptr(), us
    a.hidden, a.hidden_stride = out.data_ptr(), cols
    y = None
    if next_norm is not None:
        a.next, a.next_eps = _norm_code(next_norm, _NORM, "next_norm"), next_eps
        next_weight = _vector(next_weight, cols, "next_weight", device)
        next_bias = _vector(next_bias, cols, "next_bias", device)
        _put_vector(a, "next_weight", next_weight)
        _put_vector(a, "next_bias", next_bias)
        y = torch.empty(residual.shape, dtype=branch.dtype, device=device)
        a.y = y.data_ptr()
    elif next_weight is not None or next_bias is not None:
        raise ValueError("next_weight and next_bias need next_norm")
    saved = None
    if save is not None:
        saved = _new_saved()
        saved.shape, saved.dtype, saved.branch_dtype = residual.shape, residual.dtype, branch.dtype
        saved.weight, saved.bias, saved.gate = weight, bias, gate_rows
        saved.next_weight, saved.next_bias = next_weight, next_bias
        _stats(a, "post", a.post, rows, device, saved)
        _keep(a, "branch", save, u, us, rows, cols, device, saved)
        if y is not None:
            _stats(a, "next", a.next, rows, device, saved)
            _keep(a, "hidden", save, out, cols, rows, cols, device, saved)
            _keep_output(a, checkpoint_output, rows, cols, residual.shape, branch.dtype, device, saved)
        saved.args = (rows, cols, a.gates, a.post, a.next, branch_scale, residual_scale)
    with torch.cuda.device(device):
        _lib.check(_lib.lib().rf_norm_forward(a, _lib.stream_ptr()), "postnorm_residual")
    return out, y, saved


def _norm_grad(dhidden, dy, saved: NormSaved, what: str):
    a = _lib.Norm()
    a.rows, a.cols, a.gates, a.post, a.next, a.branch_scale, a.residual_scale = saved.args
    rows, cols, device, shape = a.rows, a.cols, (saved.branch if a.post else saved.hidden).device, saved.shape
    a.dtype, a.branch_dtype = _DTYPE[saved.dtype], _DTYPE[saved.branch_dtype]
    keep = []
    if dhidden is not None:
        v, a.dhidden_stride = _like(dhidden, shape, saved.dtype, "dout" if a.post else "dresidual", device)
        a.dhidden = v.data_ptr()
        keep.append(v)
    if a.next:
        if dy is None:
            raise ValueError("dy is missing")
        v, a.dy_stride = _like(dy, shape, saved.branch_dtype, "dy", device)
        a.dy = v.data_ptr()
        keep.append(v)
    elif dy is not None:
        raise ValueError("dy without a next norm")
    for part in ("post", "next"):
        rstd = getattr(saved, part + "_rstd")
        if rstd is not None:
            setattr(a, part + "_rstd", rstd.data_ptr())
            setattr(a, part + "_mean", rstd.data_ptr() + 4 * rows if rstd.numel() == 2 * rows else None)
    for name in ("branch", "hidden"):
        t, exps = getattr(saved, name), getattr(saved, name + "_exponents")
        if exps is not None:
            setattr(a, name + "_codes", t.data_ptr())
            setattr(a, name + "_exponents", exps.data_ptr())
        elif t is not None:
            setattr(a, name, t.data_ptr())
            setattr(a, name + "_stride", t.stride(0))
    grads = {}
    for name in ("weight", "bias", "gate", "next_weight", "next_bias"):
        v = getattr(saved, name)
        grads[name] = None
        if v is not None:
            _put_vector(a, name, v)
            grads[name] = torch.empty_like(v)
            setattr(a, "d" + name, grads[name].data_ptr())
    dresidual = torch.empty(shape, dtype=saved.dtype, device=device)
    a.dresidual, dbranch = dresidual.data_ptr(), None
    if a.post:
        dbranch = torch.empty(shape, dtype=saved.branch_dtype, device=device)
        a.dbranch = dbranch.data_ptr()
    with torch.cuda.device(device):
        space, size = _workspace(_lib.lib().rf_norm_backward_workspace, a, device, what)
        _lib.check(_lib.lib().rf_norm_backward(a, space, size, _lib.stream_ptr()), what)
    return dresidual, dbranch, grads


def prenorm_grad(dy, saved: NormSaved, *, dresidual=None) -> PrenormGrads:
    """Gradients of ``prenorm``'s x, weight and bias.  ``dresidual``: another
    gradient at x (the residual path's), added to x's in the same pass."""
    if saved.args[3] != _lib.RF_NORM_ABSENT:
        raise ValueError("saved is postnorm_residual's: use postnorm_residual_grad")
    dx, _, g = _norm_grad(dresidual, dy, saved, "prenorm_grad")
    return PrenormGrads(dx, g["next_weight"], g["next_bias"])


def postnorm_residual_grad(dout, dy, saved: NormSaved) -> PostnormGrads:
    """Gradients of ``postnorm_residual`` from those of out (None: zero) and,
    with a next norm, of y."""
    if saved.args[3] == _lib.RF_NORM_ABSENT:
        raise ValueError("saved is prenorm's: use prenorm_grad")
    dr, du, g = _norm_grad(dout, dy, saved, "postnorm_residual_grad")
    return PostnormGrads(dr, du, g["weight"], g["bias"], g["gate"], g["next_weight"], g["next_bias"])
