"""The loss of a language model over its vocabulary (no reference counterpart).

``linear_cross_entropy`` is the softmax cross entropy of ``hidden @ weight.T``:

    loss = lse - logit[target] + z_loss * lse ** 2,  lse = log(sum(exp(logits)))

for every row of ``hidden``; no logit is written: each tile of the product is
reduced to a maximum and a sum as it is computed.
``linear_cross_entropy_grad`` gives the gradients of ``hidden`` and ``weight`` as
well, in the same pass, and computes no product twice.  For that it holds the
exponentials of a piece of the tokens, at most 2 GiB at once: 16 bits each (up to
that size all of them, as much as 16-bit logits), float32 tensors' 32 and as much
again.
``rollfast_amd.autograd.linear_cross_entropy`` is differentiable.

A token whose target is ``ignore_index`` has a loss of zero and no part in the
gradients, whatever its row of ``hidden`` holds (its own gradient is zero).  A
target that is no row of ``weight`` otherwise makes the loss and the gradients NaN.
In float32 an Inf in ``weight`` makes every loss NaN, and one in a row of ``hidden``
its own, since split numbers have no infinities of one sign.

``hidden`` and ``weight`` are float32, bfloat16 or float16 on a ROCm device, both
of one dtype, which is the gradients' too; losses are float32.  Targets are int32
or int64.  Any row stride is read in place.  Work is enqueued on the current
stream.

Sums are f32 in a fixed order: equal inputs give equal bits.  (How they are split
follows from how many tokens count, so a token's last bits may differ from batch to
batch.)  16-bit tensors are multiplied as they are, float32 ones to 22 bits, of
which those below 2^-39 of the largest magnitude in ``hidden``, or ``weight``, are
lost.  The gradient of a logit is rounded to the tensors' own dtype (float32: to 22
bits; 16-bit ones where at most 16 tokens count: to twice its bits) before it is
multiplied.  In float16 and float32 it is held down to 2^-33 of its token's own
``dloss`` at least, however much other tokens weigh; what a token adds to the
weight's gradient is also lost below 2^-39 of what the heaviest one may add.  For
16-bit tensors exponentials are rounded to float16: a probability below 2^-25 of
the largest among its 64 or 128 neighbours in the vocabulary has no part in the
gradients.
"""

from __future__ import annotations

import ctypes
from typing import Any, NamedTuple

import torch

from . import _lib
from .blocks import _code, _rows, _tensor

_REDUCTION = {"none": _lib.RF_REDUCE_NONE, "sum": _lib.RF_REDUCE_SUM, "mean": _lib.RF_REDUCE_MEAN}


class LossGrads(NamedTuple):
    loss: Any
    hidden: Any
    weight: Any


def _arguments(hidden, weight, targets, ignore_index, z_loss, reduction):
    """The call's structure and the tensors that it points to."""
    device = _tensor(hidden, "hidden").device
    _tensor(weight, "weight", device)
    _tensor(targets, "targets", device)
    a = _lib.CrossEntropy()
    a.dtype = _code(hidden.dtype, "hidden")
    if weight.dtype != hidden.dtype:
        raise ValueError(f"weight is {weight.dtype}, hidden is {hidden.dtype}")
    if hidden.dim() == 0 or weight.dim() != 2 or weight.shape[1] != hidden.shape[-1]:
        raise ValueError(f"hidden [..., n] and weight [vocab, n] do not fit: {tuple(hidden.shape)}, {tuple(weight.shape)}")
    if weight.shape[0] == 0:
        raise ValueError("weight needs at least one row")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets have shape {tuple(targets.shape)}, expected {tuple(hidden.shape[:-1])}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"targets must be int64 or int32, got {targets.dtype}")
    if reduction not in _REDUCTION:
        raise ValueError(f"reduction must be one of {', '.join(map(repr, _REDUCTION))}, got {reduction!r}")
    rows, hidden_stride = _rows(hidden, "hidden")
    table, weight_stride = _rows(weight, "weight")
    targets = targets.contiguous()
    a.tokens, a.vocab, a.hidden = targets.numel(), weight.shape[0], weight.shape[1]
    a.target_bits = 64 if targets.dtype == torch.int64 else 32
    a.hidden_rows, a.weight, a.targets = rows.data_ptr(), table.data_ptr(), targets.data_ptr()
    a.hidden_stride, a.weight_stride = hidden_stride, weight_stride
    a.ignore_index, a.z_loss, a.reduction = int(ignore_index), float(z_loss), _REDUCTION[reduction]
    return a, (rows, table, targets)


def _call(hidden, weight, targets, dloss, ignore_index, z_loss, reduction, grad, wide=False):
    """(loss, dhidden, dweight): the native host path where the tensors are as
    they may be, on the current device; else laid out here.  ``wide``: the
    gradients in float32, whatever the tensors are."""
    code = _REDUCTION.get(reduction)
    if code is not None:
        code |= _lib.RF_GRADS_F32 if wide else 0
        got = _lib.pyblocks().cross_entropy(hidden, weight, targets, dloss, int(ignore_index), float(z_loss), code, grad)
        if got is not None:
            return got
    a, _held = _arguments(hidden, weight, targets, ignore_index, z_loss, reduction)
    device = hidden.device
    if dloss is not None:
        _tensor(dloss, "dloss", device)
        if dloss.shape != targets.shape or dloss.dtype != torch.float32:
            raise ValueError(f"dloss must be float32 of shape {tuple(targets.shape)}, got {dloss.dtype} {tuple(dloss.shape)}")
        dloss = dloss.contiguous()
        a.dloss = dloss.data_ptr()
    total = dhidden = dweight = None
    with torch.cuda.device(device):
        loss = torch.empty(targets.shape, dtype=torch.float32, device=device)
        a.loss = loss.data_ptr()
        if reduction != "none":
            total = torch.empty((), dtype=torch.float32, device=device)
            a.total = total.data_ptr()
        if grad:
            dtype = torch.float32 if wide else hidden.dtype
            dhidden = torch.empty(hidden.shape, dtype=dtype, device=device)
            dweight = torch.empty(weight.shape, dtype=dtype, device=device)
            a.reduction |= _lib.RF_GRADS_F32 if wide else 0
            a.dhidden, a.dweight = dhidden.data_ptr(), dweight.data_ptr()
        need, what = ctypes.c_int64(), "linear_cross_entropy_grad" if grad else "linear_cross_entropy"
        _lib.check(_lib.lib().rf_linear_cross_entropy_workspace(a, need), what)
        workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
        _lib.check(_lib.lib().rf_linear_cross_entropy(a, workspace.data_ptr(), need.value, _lib.stream_ptr()), what)
    return loss if reduction == "none" else total, dhidden, dweight


def linear_cross_entropy(hidden, weight, targets, *, ignore_index: int = -100, z_loss: float = 0.0,
                         reduction: str = "none"):
    """The loss of every row of ``hidden`` [..., n] with ``targets`` [...] and
    ``weight`` [vocab, n], in float32: of the targets' shape, or with
    ``reduction`` 'sum' or 'mean' one value over the targets that count."""
    return _call(hidden, weight, targets, None, ignore_index, z_loss, reduction, False)[0]


def linear_cross_entropy_grad(hidden, weight, targets, dloss=None, *, ignore_index: int = -100, z_loss: float = 0.0,
                              reduction: str = "none") -> LossGrads:
    """The losses, and the gradients of ``sum(dloss * loss)`` with ``dloss``
    float32 of the targets' shape; or with a ``reduction`` in place of ``dloss``
    the reduced loss and its gradients.  float16 gradients of a mean over many
    tokens lie below float16's normal numbers: give a ``dloss`` with the scale of
    the loss in it, or take ``autograd.linear_cross_entropy``."""
    if (dloss is None) == (reduction == "none"):
        raise ValueError("the gradient needs dloss, or a reduction in its place")
    return LossGrads(*_call(hidden, weight, targets, dloss, ignore_index, z_loss, reduction, True))
