"""Refusals of the residual-block operators that need no GPU: the C entries
check their arguments before any device work, and the Python functions refuse
host tensors and bad options."""

from __future__ import annotations

import ctypes

import pytest
import torch

import rollfast_amd as rf
from rollfast_amd import _lib

P = 4096  # a pointer that is never read: every call below is refused


def refused(status, text, code=1):
    assert status == code
    assert text in _lib.lib().rf_last_error().decode()


def test_structs_match_the_header(tmp_path):
    import os
    import shutil
    import subprocess

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lines = ['#include "rfadam8.h"', "#include <stddef.h>"]
    for c, py in (("rf_norm", _lib.Norm), ("rf_gated", _lib.Gated), ("rf_weight_grad", _lib.WeightGrad)):
        lines.append(f"typedef char {c}_size[sizeof({c}) == {ctypes.sizeof(py)} ? 1 : -1];")
        lines += [f"typedef char {c}_{n}[offsetof({c}, {n}) == {getattr(py, n).offset} ? 1 : -1];" for n, _ in py._fields_]
    src = tmp_path / "s.c"
    src.write_text("\n".join(lines) + "\nint main(void) { return 0; }\n")
    r = subprocess.run([cc, "-std=c99", "-pedantic", "-Werror", "-I", os.path.join(root, "include"), "-fsyntax-only",
                        str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_checkpoint_refusals():
    L = _lib.lib()
    refused(L.rf_checkpoint_store(P, 0, -1, 4, 4, P, P, None), "out of range")
    refused(L.rf_checkpoint_store(P, 0, 4, 0, 4, P, P, None), "out of range")
    refused(L.rf_checkpoint_store(P, 7, 4, 4, 4, P, P, None), "dtype", 3)
    refused(L.rf_checkpoint_store(None, 0, 4, 4, 4, P, P, None), "null")
    refused(L.rf_checkpoint_store(P, 0, 4, 4, 4, P + 8, P, None), "aligned")
    refused(L.rf_checkpoint_load(P, P, 4, 4, 9, P, None), "dtype", 3)
    refused(L.rf_checkpoint_load(P, None, 4, 4, 0, P, None), "null")
    assert L.rf_checkpoint_store(None, 0, 0, 4, 4, None, None, None) == 0
    assert L.rf_checkpoint_load(None, None, 0, 4, 0, None, None) == 0


def gated(**over):
    a = _lib.Gated()
    a.rows, a.cols, a.gate, a.up, a.h, a.dh, a.dgate, a.dup = 4, 8, P, P, P, P, P, P
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_gated_refusals():
    L = _lib.lib()
    refused(L.rf_gated_forward(None, None), "null")
    refused(L.rf_gated_forward(gated(dtype=5), None), "dtype", 3)
    refused(L.rf_gated_forward(gated(activation=3), None), "activation")
    refused(L.rf_gated_forward(gated(cols=0), None), "out of range")
    refused(L.rf_gated_forward(gated(h=None), None), "null")
    refused(L.rf_gated_forward(gated(gate_codes=P, gate_exponents=P), None), "together")
    refused(L.rf_gated_forward(gated(gate_codes=P, up_codes=P), None), "together")
    refused(L.rf_gated_backward(gated(gate=None), None), "null")
    refused(L.rf_gated_backward(gated(dup=None), None), "null")
    assert L.rf_gated_forward(gated(rows=0), None) == 0


def norm(**over):
    a = _lib.Norm()
    a.rows, a.cols, a.post, a.next, a.branch_scale, a.residual_scale = 4, 8, 2, 2, 1.0, 1.0
    for k in ("residual", "branch", "hidden", "y", "dhidden", "dy", "dresidual", "dbranch", "post_rstd", "next_rstd"):
        setattr(a, k, P)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_norm_refusals():
    L = _lib.lib()
    refused(L.rf_norm_forward(None, None), "null")
    for over, text in (({"rows": -1}, "out of range"), ({"cols": 0}, "out of range"), ({"post": 4}, "post"),
                       ({"next": 1}, "next"), ({"post": 0, "next": 0}, "neither"), ({"gates": 3, "gate": P}, "gates"),
                       ({"gates": 2}, "gates"), ({"gate": P}, "gates"), ({"post": 0, "weight": P}, "without"),
                       ({"post": 1, "bias": P}, "without"), ({"branch_codes": P}, "together"),
                       ({"hidden_codes": P + 4, "hidden_exponents": P}, "aligned"), ({"hidden": None}, "null"),
                       ({"y": None}, "null"), ({"branch": None}, "null"), ({"post_eps": -1.0}, "eps"),
                       ({"next_eps": float("nan")}, "eps")):
        refused(L.rf_norm_forward(norm(**over), None), text)
    refused(L.rf_norm_forward(norm(dtype=1, branch_dtype=0), None), "dtype", 3)
    refused(L.rf_norm_forward(norm(weight=P, weight_dtype=9), None), "dtype", 3)
    assert L.rf_norm_forward(norm(rows=0), None) == 0
    for over, text in (({"branch_codes": P, "branch_exponents": P}, "neither"), ({"dweight": P}, "absent"),
                       ({"dgate": P}, "absent"), ({"dnext_bias": P}, "absent"), ({"dy": None}, "null"),
                       ({"dresidual": None}, "null"), ({"post_rstd": None}, "statistics"),
                       ({"next": 3}, "statistics"), ({"post": 3}, "statistics")):
        refused(L.rf_norm_backward(norm(**over), None, 0, None), text)


def test_weight_grad_refusals():
    def args(**over):
        a = _lib.WeightGrad()
        a.rows, a.outs, a.cols, a.dy, a.codes, a.exponents, a.out = 4, 8, 8, P, P, P, P
        for k, v in over.items():
            setattr(a, k, v)
        return a

    L = _lib.lib()
    refused(L.rf_linear_weight_grad(None, None, 0, None), "null")
    for over, text, code in (({"rows": -1}, "out of range", 1), ({"outs": 0}, "out of range", 1),
                             ({"cols": 0}, "out of range", 1), ({"dy_dtype": 4}, "dtype", 3),
                             ({"out_dtype": 4}, "dtype", 3), ({"codes": P + 1}, "aligned", 1), ({"out": None}, "null", 1),
                             ({"dy": None}, "null", 1), ({"exponents": None}, "null", 1)):
        refused(L.rf_linear_weight_grad(args(**over), None, 0, None), text, code)
    refused(L.rf_linear_weight_grad_workspace(args(), None), "null")


def test_python_refusals():
    x = torch.zeros(4, 8)
    for call in (lambda: rf.checkpoint_activations(x), lambda: rf.prenorm(x), lambda: rf.postnorm_residual(x, x),
                 lambda: rf.gated_activation(x, x),
                 lambda: rf.linear_weight_grad(x, rf.ActivationCheckpoint(x, x, (4, 8), x.dtype))):
        with pytest.raises(ValueError, match="ROCm device"):
            call()
    with pytest.raises(TypeError, match="torch.Tensor"):
        rf.prenorm([1.0])
    with pytest.raises(ValueError, match="save"):
        rf.prenorm(x, save="fp8")
    with pytest.raises(ValueError, match="activation"):
        rf.gated_activation(x, x, activation="relu")
    with pytest.raises(ValueError, match="checkpoint_output"):
        rf.prenorm(x, save=None, checkpoint_output=True)


@pytest.mark.gpu
def test_python_refusals_on_a_gpu():
    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    ck = rf.checkpoint_activations(x)
    _, pre = rf.prenorm(x, w)
    out, _, post = rf.postnorm_residual(x, x, w)
    _, gs = rf.gated_activation(x, x)
    bad = [
        (lambda: rf.checkpoint_activations(x[0, 0]), "last dimension"),
        (lambda: rf.checkpoint_activations(x[:, :0]), "last dimension"),
        (lambda: rf.prenorm(x, w[:5]), "shape"),
        (lambda: rf.prenorm(x, w.cpu()), "ROCm"),
        (lambda: rf.prenorm(x, w, norm="none"), "norm must be"),
        (lambda: rf.postnorm_residual(x, x[:2]), "shape"),
        (lambda: rf.postnorm_residual(x, x, w, norm="none"), "norm='none'"),
        (lambda: rf.postnorm_residual(x, x, gate=torch.ones(3, 8, device="cuda")), "gate"),
        (lambda: rf.postnorm_residual(x, x, next_weight=w), "next_norm"),
        (lambda: rf.postnorm_residual(x, x, checkpoint_output=True), "next_norm"),
        (lambda: rf.prenorm_grad(x, post), "postnorm_residual_grad"),
        (lambda: rf.postnorm_residual_grad(x, None, pre), "prenorm_grad"),
        (lambda: rf.postnorm_residual_grad(x, x, post), "without a next norm"),
        (lambda: rf.prenorm_grad(None, pre), "dy"),
        (lambda: rf.prenorm_grad(x.half(), pre), "expected"),
        (lambda: rf.prenorm_grad(x[:2], pre), "shape"),
        (lambda: rf.gated_activation(x, x.half()), "expected"),
        (lambda: rf.gated_activation(x[:, :5]), "halves"),
        (lambda: rf.gated_activation_grad(x[:3], gs), "shape"),
        (lambda: rf.linear_weight_grad(x[:3], ck), "rows differ"),
        (lambda: rf.linear_weight_grad(x, ck, accumulate=True), "accumulate needs out"),
        (lambda: rf.linear_weight_grad(x, ck, out=x), "shape"),
        (lambda: rf.linear_weight_grad(x, ck._replace(shape=(4, 40))), "codes"),
        (lambda: rf.linear_weight_grad(x, ck._replace(codes=ck.codes.float())), "int8"),
        (lambda: rf.restore_activations(ck._replace(codes=ck.codes.t().contiguous().t())), "contiguous"),
    ]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()
    for call in (lambda: rf.checkpoint_activations(x.double()), lambda: rf.prenorm(x.half(), dtype=torch.bfloat16),
                 lambda: rf.linear_weight_grad(x, ck, dtype=torch.float64), lambda: rf.prenorm(x, w.double())):
        with pytest.raises(NotImplementedError):
            call()
