"""ctypes binding of ``librfadam8.so`` (C ABI declared in ``include/rfadam8.h``).

The library is required: there is no fallback implementation.  Importing
works without a GPU (the symbols load), but every compute entry point needs
its tensors on a ROCm device and raises if the library was not built.
"""

from __future__ import annotations

import ctypes
import os

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "_lib", "librfadam8.so")

RF_OK, RF_ERR_INVALID, RF_ERR_HIP, RF_ERR_UNSUPPORTED = 0, 1, 2, 3
RF_F32, RF_BF16, RF_F16 = 0, 1, 2
RF_MOMENT_QUANTIZED, RF_MOMENT_F32, RF_MOMENT_BF16, RF_MOMENT_F16 = 0, 1, 2, 3
RF_Q_DYNAMIC_SIGNED, RF_Q_DYNAMIC_UNSIGNED, RF_Q_SYMMETRIC_INT8 = 0, 1, 2
RF_NESTEROV = 1
RF_DECAY_WEAK = 4
RF_LR = 8
RF_MOMENT_SR = 16
RF_PARAM_SR = 32
RF_EXACT = 128
RF_FED_BITS = 256
RF_SKIP_NONFINITE = 512
RF_PACKED_BITS = 1024
RF_ABI_VERSION = 2
RF_LEAF_DECAY = 1
RF_LEAF_STORE_SR = 2
RF_LEAF_ZERO_DECAY = 4
RF_LEAF_SCALE_BF16 = 8
RF_LEAF_SCALE_F16 = 16
RF_ACC_SUM, RF_ACC_MEAN, RF_ACC_ZERO = 0, 1, 2
RF_NOALLOC_SCRATCH_BYTES = 8 << 20
RF_ACT_SILU, RF_ACT_GELU, RF_ACT_GELU_TANH = 0, 1, 2
RF_REDUCE_NONE, RF_REDUCE_SUM, RF_REDUCE_MEAN = 0, 1, 2
RF_GRADS_F32 = 256
RF_NORM_ABSENT, RF_NORM_NONE, RF_NORM_RMS, RF_NORM_LAYER = 0, 1, 2, 3

_p = ctypes.c_void_p


class Adam8Leaf(ctypes.Structure):
    _fields_ = [
        ("param", _p),
        ("grad", _p),
        ("updates", _p),
        ("mu", _p),
        ("mu_scales", _p),
        ("nu", _p),
        ("nu_scales", _p),
        ("mu_bits", _p),
        ("nu_bits", _p),
        ("param_bits", _p),
        ("size", ctypes.c_int64),
        ("block_size", ctypes.c_int32),
        ("param_dtype", ctypes.c_int32),
        ("grad_dtype", ctypes.c_int32),
        ("moment_kind", ctypes.c_int32),
        ("state_index", ctypes.c_int32),
        ("param_index", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
        ("group", ctypes.c_int32),
    ]


class Adam8Group(ctypes.Structure):
    _fields_ = [
        ("neg_lr", ctypes.c_float),
        ("weight_decay", ctypes.c_float),
        ("one_minus_b1", ctypes.c_float),
        ("reserved", ctypes.c_uint32),
        ("key_mu", ctypes.c_uint32 * 2),
        ("key_nu", ctypes.c_uint32 * 2),
    ]


class Adam8Hparams(ctypes.Structure):
    _fields_ = [
        ("b1", ctypes.c_float),
        ("one_minus_b1", ctypes.c_float),
        ("b2", ctypes.c_float),
        ("one_minus_b2", ctypes.c_float),
        ("bc1", ctypes.c_float),
        ("bc2", ctypes.c_float),
        ("bc1_next", ctypes.c_float),
        ("eps", ctypes.c_float),
        ("eps_root", ctypes.c_float),
        ("weight_decay", ctypes.c_float),
        ("neg_lr", ctypes.c_float),
        ("flags", ctypes.c_uint32),
        ("key_mu", ctypes.c_uint32 * 2),
        ("key_nu", ctypes.c_uint32 * 2),
        ("key_param", ctypes.c_uint32 * 2),
        ("nesterov_one_minus_b1", ctypes.c_float),
        ("clip_max_norm", ctypes.c_float),
        ("clip_out", _p),
        ("finite_out", _p),
        ("finite_host", _p),
        ("groups", _p),
        ("n_groups", ctypes.c_int32),
        ("reserved0", ctypes.c_int32),
        ("magma_sums", _p),
    ]


class ClipLeaf(ctypes.Structure):
    _fields_ = [
        ("grad", _p),
        ("out", _p),
        ("size", ctypes.c_int64),
        ("dtype", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


class MagmaLeaf(ctypes.Structure):
    _fields_ = [
        ("grad", _p),
        ("mu", _p),
        ("updates", _p),
        ("size", ctypes.c_int64),
        ("grad_dtype", ctypes.c_int32),
        ("mu_dtype", ctypes.c_int32),
        ("key_index", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


class AccumLeaf(ctypes.Structure):
    _fields_ = [
        ("grad", _p),
        ("acc", _p),
        ("size", ctypes.c_int64),
        ("grad_dtype", ctypes.c_int32),
        ("acc_dtype", ctypes.c_int32),
    ]


class ApplyLeaf(ctypes.Structure):
    _fields_ = [
        ("param", _p),
        ("updates", _p),
        ("bits", _p),
        ("size", ctypes.c_int64),
        ("param_dtype", ctypes.c_int32),
        ("param_index", ctypes.c_int32),
    ]


_i32, _i64, _f32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class Gated(ctypes.Structure):
    _fields_ = [
        *((n, _i64) for n in ("rows", "cols")),
        *((n, _i32) for n in ("dtype", "activation")),
        *((n, _p) for n in ("gate", "up")),
        *((n, _i64) for n in ("gate_stride", "up_stride")),
        *((n, _p) for n in ("gate_codes", "gate_exponents", "up_codes", "up_exponents", "h", "h_codes", "h_exponents",
                            "dh")),
        ("dh_stride", _i64),
        *((n, _p) for n in ("dgate", "dup")),
        *((n, _i64) for n in ("dgate_stride", "dup_stride")),
    ]


class Norm(ctypes.Structure):
    _fields_ = [
        *((n, _i64) for n in ("rows", "cols", "gates")),
        *((n, _i32) for n in ("dtype", "branch_dtype", "post", "next")),
        *((n, _f32) for n in ("post_eps", "next_eps", "branch_scale", "residual_scale")),
        *((n, _p) for n in ("residual", "branch", "hidden")),
        *((n, _i64) for n in ("residual_stride", "branch_stride", "hidden_stride")),
        *((n, _p) for n in ("weight", "bias", "gate", "next_weight", "next_bias")),
        *((n, _i32) for n in ("weight_dtype", "bias_dtype", "gate_dtype", "next_weight_dtype", "next_bias_dtype",
                              "reserved")),
        *((n, _p) for n in ("y", "branch_codes", "branch_exponents", "hidden_codes", "hidden_exponents", "y_codes",
                            "y_exponents", "post_mean", "post_rstd", "next_mean", "next_rstd", "dhidden", "dy")),
        *((n, _i64) for n in ("dhidden_stride", "dy_stride")),
        *((n, _p) for n in ("dresidual", "dbranch", "dweight", "dbias", "dgate", "dnext_weight", "dnext_bias")),
    ]


class WeightGrad(ctypes.Structure):
    _fields_ = [
        *((n, _i64) for n in ("rows", "outs", "cols")),
        *((n, _i32) for n in ("dy_dtype", "out_dtype")),
        ("dy", _p),
        ("dy_stride", _i64),
        *((n, _p) for n in ("codes", "exponents", "out")),
        *((n, _i32) for n in ("accumulate", "reserved")),
    ]


class CrossEntropy(ctypes.Structure):
    _fields_ = [
        *((n, _i64) for n in ("tokens", "vocab", "hidden")),
        *((n, _i32) for n in ("dtype", "target_bits")),
        *((n, _p) for n in ("hidden_rows", "weight")),
        *((n, _i64) for n in ("hidden_stride", "weight_stride")),
        ("targets", _p),
        ("ignore_index", _i64),
        *((n, _p) for n in ("loss", "total", "dloss", "dhidden", "dweight")),
        ("z_loss", ctypes.c_float),
        ("reduction", _i32),
    ]


class OrthogonalMatrix(ctypes.Structure):
    _fields_ = [
        *((n, _p) for n in ("in_", "out")),
        *((n, _i64) for n in ("rows", "cols", "in_stride", "out_stride")),
        ("dtype", _i32),
        ("scale", ctypes.c_float),
    ]


class Muon8Leaf(ctypes.Structure):
    _fields_ = [
        *((n, _p) for n in ("grad", "update", "param", "codes", "scales", "momentum")),
        *((n, _i64) for n in ("rows", "cols")),
        *((n, _i32) for n in ("block_size", "dtype", "param_dtype")),
        *((n, ctypes.c_float) for n in ("scale", "decay")),
        ("reserved", _i32),
    ]


assert ctypes.sizeof(Adam8Leaf) == 120
assert ctypes.sizeof(Adam8Hparams) == 128
assert ctypes.sizeof(Adam8Group) == 32
assert ctypes.sizeof(ApplyLeaf) == 40
assert ctypes.sizeof(ClipLeaf) == 32
assert ctypes.sizeof(AccumLeaf) == 32

# Every symbol the header declares (checked by the CPU test suite).
EXPORTS = (
    "rf_adam8_plan_create",
    "rf_adam8_plan_run",
    "rf_adam8_plan_run_leaves",
    "rf_adam8_plan_wait_prepass",
    "rf_adam8_plan_info",
    "rf_adam8_plan_stream_probe",
    "rf_adam8_plan_destroy",
    "rf_adam8_step",
    "rf_adam8_step_noalloc",
    "rf_blockwise_quantize",
    "rf_blockwise_dequantize",
    "rf_sr_bf16",
    "rf_sr_bf16_packed",
    "rf_apply_updates",
    "rf_apply_updates_packed",
    "rf_clip_by_global_norm",
    "rf_all_finite",
    "rf_magma_reduce",
    "rf_magma_scale",
    "rf_magma_apply_updates",
    "rf_accumulate",
    "rf_checkpoint_store",
    "rf_checkpoint_load",
    "rf_gated_forward",
    "rf_gated_backward",
    "rf_norm_forward",
    "rf_norm_backward_workspace",
    "rf_norm_backward",
    "rf_linear_weight_grad_workspace",
    "rf_linear_weight_grad",
    "rf_linear_cross_entropy_workspace",
    "rf_linear_cross_entropy",
    "rf_orthogonalize_workspace",
    "rf_orthogonalize",
    "rf_muon8_update_workspace",
    "rf_muon8_update",
    "rf_codebook",
    "rf_host_table_codes",
    "rf_host_search_index",
    "rf_host_sr_records",
    "rf_version",
    "rf_abi_version",
    "rf_last_error",
)

_lib = None


class LibraryMissing(RuntimeError):
    pass


def lib() -> ctypes.CDLL:
    """Load (once) and return the HIP library; raises if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise LibraryMissing(
            f"{LIB_PATH} is not built; run `python -m rollfast_amd.build` "
            "(hipcc --offload-arch=gfx950) first"
        )
    L = ctypes.CDLL(LIB_PATH)
    i32, i64, u32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_uint32
    L.rf_version.restype = ctypes.c_char_p
    L.rf_last_error.restype = ctypes.c_char_p
    L.rf_adam8_plan_create.argtypes = [ctypes.POINTER(Adam8Leaf), i32, i32, ctypes.POINTER(_p)]
    L.rf_adam8_plan_run.argtypes = [_p, ctypes.POINTER(Adam8Hparams), _p]
    L.rf_adam8_plan_run_leaves.argtypes = [_p, ctypes.POINTER(Adam8Leaf), i32, ctypes.POINTER(Adam8Hparams), _p]
    L.rf_adam8_plan_info.argtypes = [_p, ctypes.POINTER(i64), ctypes.POINTER(i64), ctypes.POINTER(i64)]
    L.rf_adam8_plan_stream_probe.argtypes = [_p, _p, ctypes.POINTER(i64)]
    L.rf_adam8_plan_destroy.argtypes = [_p]
    L.rf_adam8_step.argtypes = [ctypes.POINTER(Adam8Leaf), i32, i32, ctypes.POINTER(Adam8Hparams), _p]
    L.rf_adam8_step_noalloc.argtypes = [ctypes.POINTER(Adam8Leaf), i32, i32, ctypes.POINTER(Adam8Hparams), _p]
    L.rf_blockwise_quantize.argtypes = [i32, _p, i32, i64, i32, i32, u32, u32, _p, _p, _p, i32, _p]
    L.rf_blockwise_dequantize.argtypes = [i32, _p, _p, i32, i64, i32, i32, _p, _p]
    L.rf_sr_bf16.argtypes = [_p, i64, u32, u32, _p, _p, _p]
    L.rf_apply_updates.argtypes = [ctypes.POINTER(ApplyLeaf), i32, i32, u32, u32, _p]
    L.rf_sr_bf16_packed.argtypes = [_p, i64, u32, u32, _p, _p]
    L.rf_apply_updates_packed.argtypes = [ctypes.POINTER(ApplyLeaf), i32, u32, u32, _p]
    f32 = ctypes.c_float
    L.rf_magma_reduce.argtypes = [ctypes.POINTER(MagmaLeaf), i32, f32, f32, _p, _p]
    L.rf_magma_scale.argtypes = [ctypes.POINTER(MagmaLeaf), i32, _p, _p, f32, f32, u32, u32, i32, f32, _p, _p]
    L.rf_magma_apply_updates.argtypes = [ctypes.POINTER(ApplyLeaf), i32, _p, f32, i32, u32, u32, _p]
    L.rf_accumulate.argtypes = [ctypes.POINTER(AccumLeaf), i32, i32, i32, _p]
    L.rf_checkpoint_store.argtypes = [_p, i32, i64, i64, i64, _p, _p, _p]
    L.rf_checkpoint_load.argtypes = [_p, _p, i64, i64, i32, _p, _p]
    L.rf_gated_forward.argtypes = [ctypes.POINTER(Gated), _p]
    L.rf_gated_backward.argtypes = [ctypes.POINTER(Gated), _p]
    L.rf_norm_forward.argtypes = [ctypes.POINTER(Norm), _p]
    L.rf_norm_backward_workspace.argtypes = [ctypes.POINTER(Norm), ctypes.POINTER(i64)]
    L.rf_norm_backward.argtypes = [ctypes.POINTER(Norm), _p, i64, _p]
    L.rf_linear_weight_grad_workspace.argtypes = [ctypes.POINTER(WeightGrad), ctypes.POINTER(i64)]
    L.rf_linear_weight_grad.argtypes = [ctypes.POINTER(WeightGrad), _p, i64, _p]
    L.rf_linear_cross_entropy_workspace.argtypes = [ctypes.POINTER(CrossEntropy), ctypes.POINTER(i64)]
    L.rf_linear_cross_entropy.argtypes = [ctypes.POINTER(CrossEntropy), _p, i64, _p]
    L.rf_orthogonalize_workspace.argtypes = [ctypes.POINTER(OrthogonalMatrix), i32, ctypes.POINTER(i64)]
    L.rf_orthogonalize.argtypes = [ctypes.POINTER(OrthogonalMatrix), i32, i32, _p, ctypes.c_float, _p, i64, _p]
    L.rf_muon8_update_workspace.argtypes = [ctypes.POINTER(Muon8Leaf), i32, ctypes.POINTER(i64)]
    L.rf_muon8_update.argtypes = [ctypes.POINTER(Muon8Leaf), i32, ctypes.c_float, ctypes.c_float, i32, i32, _p,
                                  ctypes.c_float, _p, i64, _p]
    L.rf_all_finite.argtypes = [ctypes.POINTER(ClipLeaf), i32, _p, _p]
    L.rf_codebook.argtypes = [i32, _p]
    L.rf_host_table_codes.argtypes = [i32, u32, i64, _p]
    L.rf_host_search_index.argtypes = [i32, u32, i64, _p]
    L.rf_host_sr_records.argtypes = [i32, _p]
    for name in EXPORTS:
        if name not in ("rf_version", "rf_last_error"):
            getattr(L, name).restype = i32
    if L.rf_abi_version() != RF_ABI_VERSION:
        raise LibraryMissing(f"{LIB_PATH} has ABI revision {L.rf_abi_version()}, this binding is written for "
                             f"{RF_ABI_VERSION}; rebuild with `python -m rollfast_amd.build`")
    _lib = L
    return L


_pyhost = None
_pyblocks = None


def _host_module(name: str):
    import importlib.util
    import sysconfig

    path = os.path.join(os.path.dirname(LIB_PATH), name + sysconfig.get_config_var("EXT_SUFFIX"))
    if not os.path.exists(path):
        raise LibraryMissing(f"{path} is not built; run `python -m rollfast_amd.build` first")
    spec = importlib.util.spec_from_file_location("rollfast_amd._lib." + name, path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def pyhost():
    """The native host fast-path module ``_rfhost`` (built with the library
    by ``rollfast_amd.build``); raises if it is not built."""
    global _pyhost
    if _pyhost is None:
        from ._base import MaskedNode

        mod = _host_module("_rfhost")
        mod.set_masked_node_type(MaskedNode)
        _pyhost = mod
    return _pyhost


def pyblocks():
    """The native host module ``_rfblocks`` of the residual-block operators
    and the vocabulary loss (built with the library by ``rollfast_amd.build``)."""
    global _pyblocks
    if _pyblocks is None:
        import torch

        L = lib()
        mod = _host_module("_rfblocks")
        names = [n for n in EXPORTS if n.startswith(("rf_checkpoint_", "rf_gated_", "rf_norm_", "rf_linear_"))]
        mod.set_entries({n: ctypes.cast(getattr(L, n), _p).value for n in (*names, "rf_last_error")},
                        torch._C._cuda_getCurrentRawStream, torch.nn.Parameter)
        _pyblocks = mod
    return _pyblocks


def check(status: int, what: str) -> None:
    """Map an rf_status to the reference's exception types."""
    if status == RF_OK:
        return
    msg = lib().rf_last_error().decode(errors="replace")
    text = f"{what}: {msg}"
    if status == RF_ERR_INVALID:
        raise ValueError(text)
    if status == RF_ERR_UNSUPPORTED:
        raise NotImplementedError(text)
    raise RuntimeError(text)


def version() -> str:
    return lib().rf_version().decode()


def codebook(signed: bool) -> np.ndarray:
    out = np.empty(256, dtype=np.float32)
    q = RF_Q_DYNAMIC_SIGNED if signed else RF_Q_DYNAMIC_UNSIGNED
    check(lib().rf_codebook(q, out.ctypes.data_as(_p)), "rf_codebook")
    return out


def host_table_codes(quantizer: int, first_bits: int, count: int) -> np.ndarray:
    out = np.empty(int(count), dtype=np.uint8)
    check(lib().rf_host_table_codes(quantizer, int(first_bits), int(count), out.ctypes.data_as(_p)),
          "rf_host_table_codes")
    return out


def host_search_index(quantizer: int, first_bits: int, count: int) -> np.ndarray:
    out = np.empty(int(count), dtype=np.uint16)
    check(lib().rf_host_search_index(quantizer, int(first_bits), int(count), out.ctypes.data_as(_p)),
          "rf_host_search_index")
    return out


def host_sr_records(quantizer: int) -> np.ndarray:
    """The moment-SR neighbour records [256, 4] (cb[li], gap, RN(1/gap) or
    0, 0) of a dynamic codebook."""
    out = np.empty((256, 4), dtype=np.float32)
    check(lib().rf_host_sr_records(quantizer, out.ctypes.data_as(_p)), "rf_host_sr_records")
    return out


def stream_ptr(device=None) -> ctypes.c_void_p:
    import torch

    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if device is None and raw is not None:  # the handle without a Stream object
        return ctypes.c_void_p(raw(torch.cuda.current_device()))
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
