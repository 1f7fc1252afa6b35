"""The residual-block operators (``rollfast_amd.blocks``) and the vocabulary loss
(``rollfast_amd.losses``) as differentiable torch functions.  What the backward pass needs is kept as 8-bit checkpoints
(``save="int8"``, the default) or as the tensors themselves
(``save="input"``); under ``torch.no_grad`` nothing is kept.

A block of a model::

    y, kept = autograd.prenorm(x, w_in, checkpoint_output=True)
    gate_up = autograd.linear(y, w_gate_up, checkpoint=kept)
    h, kept = autograd.gated_activation(gate_up, checkpoint_output=True)
    branch = autograd.linear(h, w_down, checkpoint=kept)
    x, y, kept = autograd.postnorm_residual(x, branch, w_out, gate=layer_scale, next_norm="rms",
                                            next_weight=w_in_2, checkpoint_output=True)
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import blocks, losses
from .blocks import ActivationCheckpoint


def _wanted(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _check_save(save):
    if save not in ("int8", "input"):
        raise ValueError(f"save must be 'int8' or 'input' where a gradient is wanted, got {save!r}")


def _stash(ctx, saved, out=None):
    """Moves saved's tensors to save_for_backward (which also notices a write
    to one of them before the backward pass).  ``out``: the output whose rows
    ``hidden_rows`` are.  It is saved itself: a view would hold the output, the
    output its graph, and the graph the view, so that an output dropped without
    a backward pass would never be freed."""
    ctx.set_materialize_grads(False)  # no zeros for the checkpoint's buffers
    vectors = getattr(saved, "vectors", ())
    rows = [n for n in saved.__slots__ if n == "arena" or n.endswith("_rows")]
    if out is not None and saved.hidden_rows is not None:
        saved.hidden_rows = out
    ctx.save_for_backward(*vectors, *(getattr(saved, n) for n in rows))
    ctx.rest = {n: getattr(saved, n) for n in saved.__slots__ if n not in rows and n not in ("vectors", "output")}
    ctx.rows, ctx.kind = rows, type(saved)


def _unstash(ctx):
    saved = ctx.kind()
    for name, value in ctx.rest.items():
        setattr(saved, name, value)
    tensors = ctx.saved_tensors
    vectors = len(tensors) - len(ctx.rows)
    if vectors:
        saved.vectors = tensors[:vectors]
    for name, value in zip(ctx.rows, tensors[vectors:]):
        setattr(saved, name, value)
    saved.output = None  # the next layer's, not this one's
    return saved


def _with_output(ctx, outputs, saved):
    """Appends the output checkpoint's buffers, or None."""
    kept = saved.output
    pair = (None, None) if kept is None else (kept.codes, kept.exponents)
    if kept is not None:
        ctx.mark_non_differentiable(*pair)
    return (*outputs, *pair)


def _checkpoint(codes, exponents, like):
    return ActivationCheckpoint(codes, exponents, tuple(like.shape), like.dtype)


class _Prenorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, options):
        y, saved = blocks.prenorm(x, weight, bias, **options)
        _stash(ctx, saved)
        return _with_output(ctx, (y,), saved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, *_):
        if dy is None:  # what used y gave no gradient
            return (None,) * 4
        return (*blocks.prenorm_grad(dy, _unstash(ctx)), None)


def prenorm(x, weight=None, bias=None, *, norm="rms", eps=1e-6, dtype=None, save="int8", checkpoint_output=False):
    """``blocks.prenorm``, differentiable -> y, or (y, its checkpoint) with
    ``checkpoint_output``."""
    options = {"norm": norm, "eps": eps, "dtype": dtype}
    if not _wanted(x, weight, bias):
        y = blocks.prenorm(x, weight, bias, save=None, **options)[0]
        return (y, None) if checkpoint_output else y
    _check_save(save)
    y, codes, exps = _Prenorm.apply(x, weight, bias, {**options, "save": save, "checkpoint_output": checkpoint_output})
    return (y, _checkpoint(codes, exps, y)) if checkpoint_output else y


class _Postnorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, weight, bias, gate, next_weight, next_bias, options):
        out, y, saved = blocks.postnorm_residual(residual, branch, weight, bias, gate, next_weight=next_weight,
                                                 next_bias=next_bias, **options)
        _stash(ctx, saved, out)
        return _with_output(ctx, (out, y), saved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dy, *_):
        if dout is None and dy is None:
            return (None,) * 8
        saved = _unstash(ctx)
        if dy is None and saved.meta[2]:  # y was not used
            dy = torch.zeros(saved.shape, dtype=saved.branch_dtype, device=saved.arena.device)
        g = blocks.postnorm_residual_grad(dout, dy, saved)
        return (g.residual, g.branch, g.weight, g.bias, g.gate, g.next_weight, g.next_bias, None)


def postnorm_residual(residual, branch, weight=None, bias=None, gate=None, *, norm="rms", eps=1e-6, branch_scale=1.0,
                      residual_scale=1.0, next_norm=None, next_weight=None, next_bias=None, next_eps=1e-6, save="int8",
                      checkpoint_output=False):
    """``blocks.postnorm_residual``, differentiable -> out; (out, y) with
    ``next_norm``; (out, y, y's checkpoint) with ``checkpoint_output``."""
    options = {"norm": norm, "eps": eps, "branch_scale": branch_scale, "residual_scale": residual_scale,
               "next_norm": next_norm, "next_eps": next_eps}
    if not _wanted(residual, branch, weight, bias, gate, next_weight, next_bias):
        out, y, _ = blocks.postnorm_residual(residual, branch, weight, bias, gate, next_weight=next_weight,
                                             next_bias=next_bias, save=None, **options)
        kept = None
    else:
        _check_save(save)
        options |= {"save": save, "checkpoint_output": checkpoint_output}
        out, y, codes, exps = _Postnorm.apply(residual, branch, weight, bias, gate, next_weight, next_bias, options)
        kept = None if codes is None else _checkpoint(codes, exps, y)
    if next_norm is None:
        return out
    return (out, y, kept) if checkpoint_output else (out, y)


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, options):
        h, saved = blocks.gated_activation(gate, up, **options)
        _stash(ctx, saved)
        return _with_output(ctx, (h,), saved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, *_):
        if dh is None:
            return (None,) * 3
        saved = _unstash(ctx)
        grads = blocks.gated_activation_grad(dh, saved)
        return (grads, None, None) if saved.fused else (*grads, None)


def gated_activation(gate, up=None, *, activation="silu", save="int8", checkpoint_output=False):
    """``blocks.gated_activation``, differentiable -> h, or (h, its
    checkpoint) with ``checkpoint_output``."""
    if not _wanted(gate, up):
        h = blocks.gated_activation(gate, up, activation=activation, save=None)[0]
        return (h, None) if checkpoint_output else h
    _check_save(save)
    h, codes, exps = _Gated.apply(gate, up, {"activation": activation, "save": save,
                                             "checkpoint_output": checkpoint_output})
    return (h, _checkpoint(codes, exps, h)) if checkpoint_output else h


def _product(x, weight, bias):
    """torch's linear with autocast's casts, but without its cache: that keeps a
    weight's for the rest of the region, and one made inside a Function's
    forward pass has no graph."""
    device = x.device.type
    if not torch.is_autocast_enabled(device):
        return torch.nn.functional.linear(x, weight, bias)
    dtype = torch.get_autocast_dtype(device)
    with torch.autocast(device, enabled=False):
        return torch.nn.functional.linear(*(t if t is None or t.dtype == torch.float64 else t.to(dtype)
                                            for t in (x, weight, bias)))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, checkpoint):
        ctx.has_bias = bias is not None
        ctx.shape, ctx.dtype = tuple(x.shape), x.dtype
        kept = (None, None)
        if ctx.needs_input_grad[1]:
            kept = blocks.checkpoint_activations(x) if checkpoint is None else checkpoint
            if tuple(kept.shape) != ctx.shape:
                raise ValueError(f"the checkpoint stands for {tuple(kept.shape)}, x has shape {ctx.shape}")
        ctx.save_for_backward(weight, kept[0], kept[1])
        return _product(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, codes, exps = ctx.saved_tensors
        dx = dw = db = None
        flat = dy.reshape(-1, dy.shape[-1])
        if ctx.needs_input_grad[0]:  # in the product's dtype, which autocast may have chosen
            dx = (flat @ weight.to(dy.dtype)).view(ctx.shape).to(ctx.dtype)
        if ctx.needs_input_grad[1]:
            dw = blocks.linear_weight_grad(dy, ActivationCheckpoint(codes, exps, ctx.shape, ctx.dtype),
                                           dtype=weight.dtype)
        if ctx.has_bias and ctx.needs_input_grad[2]:
            db = flat.sum(0)
        return dx, dw, db, None


def linear(x, weight, bias=None, *, checkpoint=None):
    """``x @ weight.T + bias`` whose weight gradient reads x from 8 bits:
    from ``checkpoint`` where one was made with x, else from one made here.
    The products with the weight are the library's, under autocast in its
    dtype; the weight's gradient has the weight's."""
    if not _wanted(x, weight, bias):
        return torch.nn.functional.linear(x, weight, bias)
    return _Linear.apply(x, weight, bias, checkpoint)


class _CrossEntropy(torch.autograd.Function):
    """Keeps the gradients of a loss' gradient of one, which the backward pass
    multiplies: of float16 tensors in float32, since those of a mean over many
    tokens are below float16's normal numbers until a loss scale has reached them."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, z_loss, reduction):
        loss, dhidden, dweight = losses._call(hidden, weight, targets, None, ignore_index, z_loss, reduction, True,
                                              wide=hidden.dtype == torch.float16)
        ctx.dtype = hidden.dtype
        ctx.save_for_backward(*(g if wanted else None for g, wanted in zip((dhidden, dweight), ctx.needs_input_grad)))
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        # a tensor of one dimension, so that the product is f32 (one of none would go to g's
        # type first: 2^16 is no f16, a third off by 2^-9 in bf16) and rounded once
        dloss = dloss.reshape(1)
        return (*(None if g is None else torch.mul(g, dloss, out=torch.empty_like(g, dtype=ctx.dtype))
                  for g in ctx.saved_tensors), None, None, None, None)


def linear_cross_entropy(hidden, weight, targets, *, ignore_index=-100, z_loss=0.0, reduction="mean"):
    """``losses.linear_cross_entropy`` summed ('sum') or averaged ('mean') over
    the targets that count, differentiable.  The forward pass computes both
    gradients in the same pass as the loss and keeps them, float16 tensors' in
    float32 and others in their own dtype; the backward pass multiplies them by
    the loss' own, a loss scale included.  Under autocast both tensors go to its
    dtype.  A mean over no targets is NaN with gradients of zero."""
    if reduction not in ("sum", "mean"):
        raise ValueError(f"reduction must be 'sum' or 'mean', got {reduction!r}")
    device = hidden.device.type
    if torch.is_autocast_enabled(device):
        dtype = torch.get_autocast_dtype(device)
        hidden, weight = hidden.to(dtype), weight.to(dtype)
    if not _wanted(hidden, weight):
        return losses.linear_cross_entropy(hidden, weight, targets, ignore_index=ignore_index, z_loss=z_loss,
                                           reduction=reduction)
    return _CrossEntropy.apply(hidden, weight, targets, ignore_index, z_loss, reduction)
