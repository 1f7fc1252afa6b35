"""Refusals of the vocabulary loss that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import rollfast_amd as rf
from rollfast_amd import _lib, autograd

P = 4096  # a pointer that is never read: every call below is refused


def refused(status, text, code=1):
    assert status == code
    assert text in _lib.lib().rf_last_error().decode()


def args(**over):
    a = _lib.CrossEntropy()
    a.tokens, a.vocab, a.hidden, a.dtype, a.target_bits = 4, 100, 64, _lib.RF_BF16, 64
    a.hidden_rows = a.weight = a.targets = a.loss = P
    a.hidden_stride = a.weight_stride = 64
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_struct_matches_the_header(tmp_path):
    import os
    import shutil
    import subprocess

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lines = ['#include "rfadam8.h"', "#include <stddef.h>"]
    for c, py in (("rf_cross_entropy", _lib.CrossEntropy), ("rf_orthogonal_matrix", _lib.OrthogonalMatrix),
                  ("rf_muon8_leaf", _lib.Muon8Leaf)):
        lines.append(f"typedef char {c}_size[sizeof({c}) == {ctypes.sizeof(py)} ? 1 : -1];")
        lines += [f"typedef char {c}_{n}[offsetof({c}, {n.rstrip('_')}) == {getattr(py, n).offset} ? 1 : -1];"
                  for n, _ in py._fields_]
    src = tmp_path / "s.c"
    src.write_text("\n".join(lines) + "\nint main(void) { return 0; }\n")
    r = subprocess.run([cc, "-std=c99", "-pedantic", "-Werror", "-I", os.path.join(root, "include"), "-fsyntax-only",
                        str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.parametrize("over,text,code", [
    ({"tokens": -1}, "out of range", 1),
    ({"tokens": 1 << 31}, "out of range", 1),
    ({"vocab": 0}, "out of range", 1),
    ({"vocab": (1 << 20) + 1}, "out of range", 1),
    ({"hidden": 0}, "out of range", 1),
    ({"hidden": (1 << 20) + 1}, "out of range", 1),
    ({"dtype": 5}, "dtype", 3),
    ({"target_bits": 16}, "int32 or int64", 3),
    ({"z_loss": -1.0}, "z_loss", 1),
    ({"z_loss": float("nan")}, "z_loss", 1),
    ({"z_loss": float("inf")}, "z_loss", 1),
    ({"hidden_stride": -1}, "negative stride", 1),
    ({"weight_stride": -64}, "negative stride", 1),
    ({"reduction": 3}, "reduction", 1),
])
def test_c_entry_refusals(over, text, code):
    L, size = _lib.lib(), ctypes.c_int64()
    refused(L.rf_linear_cross_entropy(args(**over), P, 1 << 40, None), text, code)
    refused(L.rf_linear_cross_entropy_workspace(args(**over), size), text, code)


@pytest.mark.parametrize("over,text", [
    ({"hidden_rows": None}, "null"),
    ({"weight": None}, "null"),
    ({"targets": None}, "null"),
    ({"loss": None}, "null"),
    ({"reduction": 1}, "total"),
    ({"reduction": 2, "total": P, "dloss": P}, "exclude"),
    ({"dweight": P, "dloss": P}, "gradients need"),
    ({"dhidden": P, "dloss": P}, "gradients need"),
    ({"dhidden": P, "dweight": P}, "gradients need"),
    ({"dloss": P}, "gradients need"),
])
def test_c_entry_buffer_refusals(over, text):
    refused(_lib.lib().rf_linear_cross_entropy(args(**over), P, 1 << 40, None), text)


def test_null_arguments():
    L = _lib.lib()
    refused(L.rf_linear_cross_entropy(None, None, 0, None), "null")
    refused(L.rf_linear_cross_entropy_workspace(args(), None), "null")


def test_python_refusals_on_the_host():
    h, w, t = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="ROCm device"):
        rf.linear_cross_entropy(h, w, t)
    with pytest.raises(TypeError):
        rf.linear_cross_entropy(None, w, t)
    with pytest.raises(ValueError, match="dloss, or a reduction"):
        rf.linear_cross_entropy_grad(h, w, t)
    with pytest.raises(ValueError, match="dloss, or a reduction"):
        rf.linear_cross_entropy_grad(h, w, t, t, reduction="sum")
    with pytest.raises(ValueError, match="reduction must be"):
        autograd.linear_cross_entropy(h, w, t, reduction="none")


@pytest.mark.gpu
def test_python_refusals():
    h, w, t = torch.zeros(4, 8, device="cuda"), torch.zeros(10, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    d = torch.zeros(4, device="cuda")
    for bad, text in (((h, w.to(torch.bfloat16), t), "weight is"), ((h, w[:, :7], t), "do not fit"), ((h, w[0], t), "do not fit"),
                      ((h, w[:0], t), "one row"), ((h, w, t[:3]), "targets have shape"), ((h, w, t.float()), "int64 or int32"),
                      ((h, w.cpu(), t), "ROCm device"), ((h, w, t.cpu()), "ROCm device"), ((h.sum(), w, t), "do not fit")):
        with pytest.raises(ValueError, match=text):
            rf.linear_cross_entropy(*bad)
    with pytest.raises(NotImplementedError):
        rf.linear_cross_entropy(h.double(), w.double(), t)
    with pytest.raises(ValueError, match="reduction must be"):
        rf.linear_cross_entropy(h, w, t, reduction="max")
    for bad in (d[:3], d.double(), d.cpu()):
        with pytest.raises(ValueError):
            rf.linear_cross_entropy_grad(h, w, t, bad)
    with pytest.raises(ValueError, match="z_loss"):
        rf.linear_cross_entropy(h, w, t, z_loss=-1.0)


def test_f32_gradients_are_added_to_a_reduction():
    L, size = _lib.lib(), ctypes.c_int64()
    for bad in (_lib.RF_GRADS_F32 | 3, _lib.RF_GRADS_F32 * 2, _lib.RF_GRADS_F32 * 2 + 1):
        refused(L.rf_linear_cross_entropy_workspace(args(reduction=bad), size), "unknown reduction")
    wide = {"dhidden": P, "dweight": P, "reduction": _lib.RF_GRADS_F32}
    refused(L.rf_linear_cross_entropy(args(**wide), P, 1 << 40, None), "gradients need")
    wide["reduction"] |= _lib.RF_REDUCE_MEAN
    refused(L.rf_linear_cross_entropy(args(**wide), P, 1 << 40, None), "total")
    refused(L.rf_linear_cross_entropy(args(**wide, total=P, dloss=P), P, 1 << 40, None), "exclude")
