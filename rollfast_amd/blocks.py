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

import math
from typing import Any, NamedTuple, Optional

import torch

from . import _lib

BLOCK = 32  # columns that share a step

_DTYPE = {torch.float32: _lib.RF_F32, torch.bfloat16: _lib.RF_BF16, torch.float16: _lib.RF_F16}
_NORM = {"rms": _lib.RF_NORM_RMS, "layer": _lib.RF_NORM_LAYER}
_POST = {"none": _lib.RF_NORM_NONE, **_NORM}
_ACT = {"silu": _lib.RF_ACT_SILU, "gelu": _lib.RF_ACT_GELU, "gelu_tanh": _lib.RF_ACT_GELU_TANH}
_SAVE = {None: 0, "int8": 1, "input": 2}


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


class _Saved:
    """What a backward pass needs.  ``arena``: one byte tensor with the codes
    of each kept row tensor, their exponents and, 16-byte aligned, the f32
    statistics; ``output``: the checkpoint of the forward pass's output, if one
    was asked for."""

    __slots__ = ()

    def _kept(self, index: int, count: int):
        """(codes, exponents) of the arena's checkpoint `index` of `count`."""
        rows, blocks = math.prod(self.shape[:-1]), -(-self.shape[-1] // BLOCK)
        codes = rows * blocks * BLOCK
        at = count * codes + index * rows * blocks
        return (self.arena[index * codes: (index + 1) * codes].view(torch.int8).view(rows, blocks * BLOCK),
                self.arena[at: at + rows * blocks].view(rows, blocks))


class NormSaved(_Saved):
    """What ``prenorm_grad`` / ``postnorm_residual_grad`` need."""

    # meta: gates, post, next, branch_scale, residual_scale, save
    # vectors: weight, bias, gate, next_weight, next_bias
    __slots__ = ("shape", "dtype", "branch_dtype", "meta", "vectors", "arena", "branch_rows", "hidden_rows", "output")

    def _of(self, name: str, index: int):
        if self.meta[5] == 2:
            return (self.branch_rows if name == "branch" else self.hidden_rows), None
        present = self.meta[1:3]
        if not present[index]:
            return None, None
        return self._kept(index if present[0] else 0, sum(map(bool, present)))

    branch = property(lambda self: self._of("branch", 0)[0])
    branch_exponents = property(lambda self: self._of("branch", 0)[1])
    hidden = property(lambda self: self._of("hidden", 1)[0])
    hidden_exponents = property(lambda self: self._of("hidden", 1)[1])


class GatedSaved(_Saved):
    """What ``gated_activation_grad`` needs."""

    __slots__ = ("activation", "shape", "dtype", "fused", "arena", "gate_rows", "up_rows", "output")


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


def _check_save(save, checkpoint_output: bool) -> int:
    mode = _SAVE.get(save)
    if mode is None:
        raise ValueError(f"save must be 'int8', 'input' or None, got {save!r}")
    if checkpoint_output and not mode:
        raise ValueError("checkpoint_output needs save='int8' or 'input'")
    return mode


def _norm_code(norm, table, what: str) -> int:
    if norm not in table:
        raise ValueError(f"{what} must be one of {', '.join(map(repr, table))}, got {norm!r}")
    return table[norm]


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


def _host():
    return _lib.pyblocks()


def _must(got, what: str):
    if got is None:  # `saved` or a checkpoint is not what its call made, or a size is past the kernels' range
        raise ValueError(f"{what}: arguments that do not fit together, or a size out of range")
    return got


# Every call goes to the native host path first, which takes plain arguments
# (contiguous tensors of the current device) as they are and returns None for
# others.  Those are checked and laid out here, on their device, and go there
# again with the shape of the outputs.


# -------------------------------------------------------------- checkpoints ---
def checkpoint_activations(x) -> ActivationCheckpoint:
    """x in 8-bit blocks of 32 columns."""
    kept = _host().checkpoint_store(x, None)
    if kept is None:
        _tensor(x, "x")
        _code(x.dtype, "x")
        v, _ = _rows(x, "x")
        with torch.cuda.device(x.device):
            kept = _must(_host().checkpoint_store(v, tuple(x.shape)), "checkpoint_activations")
    return ActivationCheckpoint(*kept, tuple(x.shape), x.dtype)


def restore_activations(checkpoint: ActivationCheckpoint, *, dtype=None):
    """The values of a checkpoint, in its own dtype or another."""
    dtype = checkpoint.dtype if dtype is None else dtype
    _code(dtype, "output")
    _check_checkpoint(checkpoint)
    args = (checkpoint.codes, checkpoint.exponents, tuple(checkpoint.shape), dtype)
    out = _host().checkpoint_load(*args)
    if out is None:
        with torch.cuda.device(checkpoint.codes.device):
            out = _must(_host().checkpoint_load(*args), "restore_activations")
    return out


def linear_weight_grad(dy, checkpoint: ActivationCheckpoint, *, out=None, accumulate: bool = False, dtype=None):
    """The gradient of ``weight`` [outs, cols] in ``y = x @ weight.T`` from
    ``dy`` [..., outs] and the checkpoint of x [..., cols].  ``out``: written,
    or added to with ``accumulate``; else a new tensor of ``dtype`` (dy's)."""
    _tensor(dy, "dy")
    _, cols = _check_checkpoint(checkpoint, dy.device)
    if dy.dim() == 0 or tuple(dy.shape[:-1]) != tuple(checkpoint.shape[:-1]):
        raise ValueError(f"dy has shape {tuple(dy.shape)}, the checkpoint {tuple(checkpoint.shape)}: their rows differ")
    outs = dy.shape[-1]
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        if dtype is not None:
            _code(dtype, "out")
    else:
        _tensor(out, "out", dy.device)
        _code(out.dtype, "out")
        if out.shape != (outs, cols) or not out.is_contiguous():
            raise ValueError(f"out must be contiguous with shape {(outs, cols)}, got {tuple(out.shape)}")
        if dtype is not None and dtype != out.dtype:
            raise ValueError(f"out is {out.dtype}, dtype says {dtype}")
    rest = (checkpoint.codes, checkpoint.exponents, cols, out, accumulate, dtype)
    got = _host().weight_grad(dy, None, *rest)
    if got is None:
        _code(dy.dtype, "dy")
        v, stride = _rows(dy, "dy")
        if stride >= 1 << 24:  # the kernel addresses a few rows by 32 bits
            v = v.contiguous()
        with torch.cuda.device(dy.device):
            got = _must(_host().weight_grad(v, tuple(dy.shape), *rest), "linear_weight_grad")
    return got


# ---------------------------------------------------------- gated activation ---
def gated_activation(gate, up=None, *, activation: str = "silu", save: Optional[str] = "int8",
                     checkpoint_output: bool = False):
    """``h = act(gate) * up`` -> (h, saved).  Without ``up`` the gate's last
    dimension holds both, the gate first (one product's output).
    ``activation``: 'silu', 'gelu' (with the error function) or 'gelu_tanh'."""
    mode = _check_save(save, checkpoint_output)
    act = _ACT.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(map(repr, _ACT))}, got {activation!r}")
    g, u = gate, up
    got = _host().gated_forward(gate, up, None, act, mode, checkpoint_output)
    if got is None:
        _tensor(gate, "gate")
        _code(gate.dtype, "gate")
        if up is None and (gate.dim() == 0 or gate.shape[-1] == 0 or gate.shape[-1] % 2):
            raise ValueError(f"without up the gate's last dimension holds both halves, got shape {tuple(gate.shape)}")
        g, _ = _rows(gate, "gate")
        u = None if up is None else _like(up, gate.shape, gate.dtype, "up", gate.device)[0]
        with torch.cuda.device(gate.device):
            got = _must(_host().gated_forward(g, u, tuple(gate.shape), act, mode, checkpoint_output), "gated_activation")
    h, arena, codes, exps = got
    if not mode:
        return h, None
    saved = GatedSaved()
    saved.activation, saved.shape, saved.dtype, saved.fused, saved.arena = act, h.shape, h.dtype, up is None, arena
    saved.gate_rows = saved.up_rows = None
    if mode == 2:
        g = _rows(g, "gate")[0].view(-1, g.shape[-1]) if g.numel() else g.reshape(0, g.shape[-1])
        cols = h.shape[-1]
        saved.gate_rows = g[:, :cols]
        saved.up_rows = g[:, cols:] if up is None else u.view(g.shape)
    saved.output = ActivationCheckpoint(codes, exps, tuple(h.shape), h.dtype) if checkpoint_output else None
    return h, saved


def gated_activation_grad(dh, saved: GatedSaved):
    """(dgate, dup); one tensor that holds both where the forward pass took one."""
    rest = (saved.activation, saved.fused, saved.arena, saved.gate_rows, saved.up_rows)
    like = saved.gate_rows if saved.arena is None else saved.arena
    got = None
    if isinstance(dh, torch.Tensor) and dh.shape == saved.shape and dh.dtype == saved.dtype and dh.device == like.device:
        got = _host().gated_backward(dh, None, *rest)
    if got is None:
        v, _ = _like(dh, saved.shape, saved.dtype, "dh", like.device)
        with torch.cuda.device(like.device):
            got = _must(_host().gated_backward(v, tuple(saved.shape), *rest), "gated_activation_grad")
    return got


# ---------------------------------------------------------------------- norms ---
def _save_norm(got, shape, dtype, meta, vectors, branch, hidden):
    """NormSaved of a forward pass's results."""
    out, y, arena, gates, codes, exps = got
    saved = NormSaved()
    saved.shape, saved.dtype, saved.branch_dtype = shape, dtype, (y if branch is None else branch).dtype
    saved.meta, saved.vectors, saved.arena = (gates, *meta), vectors, arena
    saved.branch_rows = saved.hidden_rows = None
    if meta[4] == 2:
        cols = shape[-1]
        if branch is not None:
            saved.branch_rows = branch.reshape(branch.numel() // cols, cols)
        if y is not None:
            saved.hidden_rows = hidden.reshape(hidden.numel() // cols, cols)
    saved.output = None if codes is None else ActivationCheckpoint(codes, exps, tuple(shape), y.dtype)
    return saved


def prenorm(x, weight=None, bias=None, *, norm: str = "rms", eps: float = 1e-6, dtype=None,
            save: Optional[str] = "int8", checkpoint_output: bool = False):
    """The norm before a block -> (y, saved):
    ``y = (x - mean) / sqrt(mean((x - mean)^2) + eps) * weight + bias`` for
    norm='layer', without the means for 'rms'.  ``dtype``: y's (x's; a 16-bit
    type beside a float32 x)."""
    mode = _check_save(save, checkpoint_output)
    rest = (0, _norm_code(norm, _NORM, "norm"), 0.0, eps, 1.0, 1.0, dtype, mode, checkpoint_output)
    v, vectors = x, (None, None, None, weight, bias)
    if dtype is not None:
        _code(dtype, "y")
    got = _host().norm_forward(x, None, None, vectors, *rest)
    if got is None:
        _tensor(x, "x")
        _code(x.dtype, "x")
        v, cols = _rows(x, "x")[0], x.shape[-1]
        vectors = (None, None, None, _vector(weight, cols, "weight", x.device), _vector(bias, cols, "bias", x.device))
        with torch.cuda.device(x.device):
            got = _must(_host().norm_forward(v, None, tuple(x.shape), vectors, *rest), "prenorm")
    if not mode:
        return got[1], None
    return got[1], _save_norm(got, x.shape, x.dtype, (*rest[:2], 1.0, 1.0, mode), vectors, None, v)


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
    mode = _check_save(save, checkpoint_output)
    post = _norm_code(norm, _POST, "norm")
    follows = 0 if next_norm is None else _norm_code(next_norm, _NORM, "next_norm")
    if not follows and (checkpoint_output or next_weight is not None or next_bias is not None):
        raise ValueError("next_weight, next_bias and checkpoint_output need next_norm")
    if post == _lib.RF_NORM_NONE and (weight is not None or bias is not None):
        raise ValueError("norm='none' takes no weight or bias")
    rest = (post, follows, eps, next_eps, branch_scale, residual_scale, None, mode, checkpoint_output)
    r, u, vectors = residual, branch, (weight, bias, gate, next_weight, next_bias)
    got = _host().norm_forward(residual, branch, None, vectors, *rest)
    if got is None:
        device = _tensor(residual, "residual").device
        _tensor(branch, "branch", device)
        _code(residual.dtype, "residual")
        _code(branch.dtype, "branch")
        r, cols = _rows(residual, "residual")[0], residual.shape[-1]
        u, _ = _like(branch, residual.shape, branch.dtype, "branch", device)
        vectors = (_vector(weight, cols, "weight", device), _vector(bias, cols, "bias", device),
                   _gates(gate, residual.shape, device)[0], _vector(next_weight, cols, "next_weight", device),
                   _vector(next_bias, cols, "next_bias", device))
        with torch.cuda.device(device):
            got = _must(_host().norm_forward(r, u, tuple(residual.shape), vectors, *rest), "postnorm_residual")
    if not mode:
        return got[0], got[1], None
    saved = _save_norm(got, residual.shape, residual.dtype, (post, follows, branch_scale, residual_scale, mode), vectors,
                       u, got[0])
    return got[0], got[1], saved


def _norm_grad(dhidden, dy, saved: NormSaved):
    post, follows = saved.meta[1:3]
    if follows and dy is None:
        raise ValueError("dy is missing")
    if not follows and dy is not None:
        raise ValueError("dy without a next norm")
    rest = (saved.vectors, saved.meta, saved.dtype, saved.branch_dtype, saved.arena, saved.branch_rows, saved.hidden_rows)
    shape, device = saved.shape, saved.arena.device
    got = None
    lead = dy if follows else dhidden
    if lead is None and not follows:
        dhidden = lead = torch.zeros(shape, dtype=saved.dtype, device=device)
    if isinstance(lead, torch.Tensor) and lead.shape == shape:
        got = _host().norm_backward(dhidden, dy, None, *rest)
    if got is None:
        if dhidden is not None:
            dhidden, _ = _like(dhidden, shape, saved.dtype, "dout" if post else "dresidual", device)
        if follows:
            dy, _ = _like(dy, shape, saved.branch_dtype, "dy", device)
        with torch.cuda.device(device):
            got = _must(_host().norm_backward(dhidden, dy, tuple(shape), *rest), "the norm's gradient")
    return got


def prenorm_grad(dy, saved: NormSaved, *, dresidual=None) -> PrenormGrads:
    """Gradients of ``prenorm``'s x, weight and bias.  ``dresidual``: another
    gradient at x (the residual path's), added to x's in the same pass."""
    if saved.meta[1] != _lib.RF_NORM_ABSENT:
        raise ValueError("saved is postnorm_residual's: use postnorm_residual_grad")
    got = _norm_grad(dresidual, dy, saved)
    return PrenormGrads(got[0], got[5], got[6])


def postnorm_residual_grad(dout, dy, saved: NormSaved) -> PostnormGrads:
    """Gradients of ``postnorm_residual`` from those of out (None: zero) and,
    with a next norm, of y."""
    if saved.meta[1] == _lib.RF_NORM_ABSENT:
        raise ValueError("saved is prenorm's: use prenorm_grad")
    return PostnormGrads(*_norm_grad(dout, dy, saved))
