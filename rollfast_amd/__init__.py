"""rollfast_amd: rollfast's 8-bit AdamW step on MI355X (gfx950) HIP kernels.

Drop-in for the reference's adam8 hot path (rollfast ``adamw8``,
``scale_by_adam8``, ``quantize_blocks``, ``dequantize_blocks``,
``apply_updates``) and its full-precision sibling (``adamw``,
``scale_by_adam``): same names, arguments, state pytree and errors, with
torch tensors on a ROCm device in place of jax arrays.  ``adamw8_step`` /
``adamw_step`` fuse ``tx.update`` and ``apply_updates`` into one HBM pass.

Beside it, without reference counterparts: the operators of a residual block with
8-bit saved activations (``blocks``), the loss over the vocabulary with its
gradients (``losses``), their differentiable forms (``autograd``), and
``orthogonalize`` with ``muon8``, the optimizer made of it.
"""

from . import prng
from ._base import (
    ApplyIfFiniteState,
    EmptyState,
    GradientTransformation,
    GradientTransformationExtraArgs,
    MaskedNode,
    MaskedState,
    ScaleByScheduleState,
)
from .optim.adam8 import (
    DYNAMIC_SIGNED_CODEBOOK_ID,
    DYNAMIC_UNSIGNED_CODEBOOK_ID,
    SYMMETRIC_INT8_CODEBOOK_ID,
    QuantizedBlocks,
    ScaleByAdam8State,
    adamw8,
    adamw8_step,
    dequantize_blocks,
    estimate_quantized_moment_bytes,
    quantize_blocks,
    quantized_nbytes,
    scale_by_adam8,
    tree_state_nbytes,
)
from .optim.adam import ScaleByAdamState, adamw, adamw_step, scale_by_adam
from .optim.convert import adam8_state_from_adam, adam_state_from_adam8, dequantize_state_tree, quantize_state_tree
from .optim.muon import Muon8State, muon8, orthogonalize
from .combine import MultiTransformState, chain, masked, multi_transform
from .transforms import GlobalNormClipState, apply_if_finite, clip_by_global_norm
from .multisteps import MultiSteps, MultiStepsState
from .utils import apply_updates, apply_updates_prefix

__version__ = "0.1.0"

# The residual-block operators (blocks.py) and their differentiable forms
# (autograd.py) import torch; the names load on first use.
_BLOCKS = (
    "ActivationCheckpoint",
    "PostnormGrads",
    "PrenormGrads",
    "checkpoint_activations",
    "gated_activation",
    "gated_activation_grad",
    "linear_weight_grad",
    "postnorm_residual",
    "postnorm_residual_grad",
    "prenorm",
    "prenorm_grad",
    "restore_activations",
)

# The vocabulary loss (losses.py), likewise.
_LOSSES = ("LossGrads", "linear_cross_entropy", "linear_cross_entropy_grad")


def __getattr__(name):
    import importlib

    if name in _BLOCKS:
        value = getattr(importlib.import_module(".blocks", __name__), name)
    elif name in _LOSSES:
        value = getattr(importlib.import_module(".losses", __name__), name)
    elif name in ("autograd", "blocks", "losses"):
        value = importlib.import_module("." + name, __name__)
    else:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    globals()[name] = value
    return value


__all__ = (
    "DYNAMIC_SIGNED_CODEBOOK_ID",
    "DYNAMIC_UNSIGNED_CODEBOOK_ID",
    "SYMMETRIC_INT8_CODEBOOK_ID",
    "ActivationCheckpoint",
    "ApplyIfFiniteState",
    "EmptyState",
    "GlobalNormClipState",
    "GradientTransformation",
    "GradientTransformationExtraArgs",
    "LossGrads",
    "MaskedNode",
    "MaskedState",
    "MultiSteps",
    "MultiStepsState",
    "MultiTransformState",
    "Muon8State",
    "PostnormGrads",
    "PrenormGrads",
    "QuantizedBlocks",
    "ScaleByAdam8State",
    "ScaleByAdamState",
    "ScaleByScheduleState",
    "adam8_state_from_adam",
    "adam_state_from_adam8",
    "adamw",
    "adamw8",
    "adamw8_step",
    "adamw_step",
    "apply_if_finite",
    "apply_updates",
    "apply_updates_prefix",
    "autograd",
    "chain",
    "checkpoint_activations",
    "clip_by_global_norm",
    "dequantize_blocks",
    "dequantize_state_tree",
    "estimate_quantized_moment_bytes",
    "gated_activation",
    "gated_activation_grad",
    "linear_cross_entropy",
    "linear_cross_entropy_grad",
    "linear_weight_grad",
    "losses",
    "masked",
    "multi_transform",
    "muon8",
    "orthogonalize",
    "postnorm_residual",
    "postnorm_residual_grad",
    "prenorm",
    "prenorm_grad",
    "prng",
    "quantize_blocks",
    "quantize_state_tree",
    "quantized_nbytes",
    "restore_activations",
    "scale_by_adam",
    "scale_by_adam8",
    "tree_state_nbytes",
)
