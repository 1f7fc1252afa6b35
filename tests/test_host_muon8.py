"""Refusals of the orthogonalisation and of muon8 that need no GPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import rollfast_amd as rf
from rollfast_amd import _lib

P = 4096  # a pointer that is never read: every call below is refused


def refused(status, text, code=1):
    assert status == code
    assert text in _lib.lib().rf_last_error().decode()


def matrix(**over):
    m = _lib.OrthogonalMatrix(P, P, 8, 16, 16, 16, _lib.RF_BF16, 1.0)
    for k, v in over.items():
        setattr(m, k, v)
    return (_lib.OrthogonalMatrix * 1)(m)


GOOD = np.tile(np.array([3.4445, -4.775, 2.0315], np.float32), (5, 1))


def call(matrices, count=1, steps=5, table=GOOD, eps=1e-7, bytes_=1 << 40, workspace=P):
    return _lib.lib().rf_orthogonalize(matrices, count, steps, None if table is None else table.ctypes.data, eps, workspace,
                                       bytes_, None)


@pytest.mark.parametrize("over,text,code", [
    ({"rows": -1}, "size out of range", 1),
    ({"cols": (1 << 20) + 1}, "size out of range", 1),
    ({"rows": 70000, "cols": 70000}, "size out of range", 1),
    ({"dtype": 9}, "dtype", 3),
    ({"in_stride": -1}, "negative stride", 1),
    ({"in_": None}, "null buffer", 1),
    ({"out": None}, "null buffer", 1),
])
def test_matrices_that_are_refused(over, text, code):
    refused(call(matrix(**over)), text, code)


def test_calls_that_are_refused():
    refused(call(matrix(), count=-1), "at most 256")
    refused(call(matrix(), count=257), "at most 256")
    refused(call(None), "at most 256")
    refused(call(matrix(), steps=-1), "steps")
    refused(call(matrix(), steps=101), "steps")
    refused(call(matrix(), table=None), "steps")
    refused(call(matrix(), eps=-1.0), "eps")
    refused(call(matrix(), eps=float("nan")), "eps")
    refused(call(matrix(), table=GOOD * np.float32("nan")), "finite")
    refused(call(matrix(), table=GOOD * 4), "grow past 64")
    refused(_lib.lib().rf_orthogonalize_workspace(matrix(), 1, None), "null")


def leaf(**over):
    x = _lib.Muon8Leaf()
    x.grad = x.update = x.codes = x.scales = P
    x.rows, x.cols, x.block_size, x.dtype = 8, 16, 256, _lib.RF_BF16
    for k, v in over.items():
        setattr(x, k, v)
    return (_lib.Muon8Leaf * 1)(x)


@pytest.mark.parametrize("over,text,code", [
    ({"rows": -1}, "size out of range", 1),
    ({"cols": (1 << 20) + 1}, "size out of range", 1),
    ({"dtype": 7}, "dtype", 3),
    ({"param": P, "param_dtype": 7}, "dtype", 3),
    ({"block_size": 0}, "block size", 1),
    ({"scales": None}, "block size", 1),
    ({"grad": None}, "null buffer", 1),
    ({"update": None}, "null buffer", 1),
    ({"codes": None}, "null buffer", 1),
])
def test_leaves_that_are_refused(over, text, code):
    refused(_lib.lib().rf_muon8_update(leaf(**over), 1, 0.9, 0.1, 1, 5, GOOD.ctypes.data, 1e-7, P, 1 << 40, None), text, code)


def test_python_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="ROCm device"):
        rf.orthogonalize(x)
    with pytest.raises(TypeError):
        rf.orthogonalize([1.0])
    for steps in (-1, 2.5, 101, True):
        with pytest.raises(ValueError, match="steps"):
            rf.orthogonalize([], steps=steps)
    for table in ((1.0, 2.0), ((1.0, 2.0, 3.0),) * 4):
        with pytest.raises(ValueError, match="coefficients"):
            rf.orthogonalize([], coefficients=table)
    for bad in ({"momentum": 1.0}, {"momentum": -0.1}, {"weight_decay": -1.0}, {"weight_decay": float("inf")}, {"block_size": 0},
                {"min_size": -1}, {"adjust": "norm"}, {"steps": -1}, {"coefficients": (1.0,)}):
        with pytest.raises(ValueError):
            rf.muon8(0.1, **bad)
    tx = rf.muon8(0.1, weight_decay=0.1)
    with pytest.raises(ValueError, match="matrices"):
        tx.init({"norm": torch.zeros(8)})
    state = rf.Muon8State(np.zeros((), np.int32), {"w": torch.zeros(4, 8)})
    with pytest.raises(ValueError, match="params"):
        tx.update({"w": x}, state)
    with pytest.raises(ValueError, match="ROCm device"):
        tx.update({"w": x}, state, {"w": x})


@pytest.mark.gpu
def test_python_refusals_on_the_device():
    x = torch.zeros(4, 8, device="cuda")
    with pytest.raises(ValueError, match="two dimensions"):
        rf.orthogonalize(x[0])
    with pytest.raises(NotImplementedError):
        rf.orthogonalize(x.double())
    with pytest.raises(ValueError, match="grow past 64"):
        rf.orthogonalize(x, coefficients=(10.0, 0.0, 0.0))
    tx = rf.muon8(0.1, weight_decay=0.1)
    state = tx.init({"w": x})
    for grads, params in (({"w": x[:3]}, {"w": x}), ({"w": x}, {"w": x[:3]}), ({"w": x.view(2, 2, 8)}, {"w": x})):
        with pytest.raises(ValueError):
            tx.update(grads, state, params)
    small = rf.muon8(0.1, min_size=0).init({"w": x})
    with pytest.raises(ValueError, match="the momentum has shape"):
        rf.muon8(0.1).update({"w": x[:3]}, small)
    other = small._replace(mu={"w": rf.quantize_blocks(x, quantizer="symmetric_int8")})
    with pytest.raises(ValueError, match="dynamic signed"):
        rf.muon8(0.1).update({"w": x}, other)


def test_finite_test_refusals():
    L = _lib.lib()
    row = _lib.ClipLeaf()
    row.grad, row.size, row.dtype = P, 8, _lib.RF_F32
    refused(L.rf_all_finite((_lib.ClipLeaf * 1)(row), 1, None, None), "null output")
    refused(L.rf_all_finite(None, 1, P, None), "bad leaf table")
    refused(L.rf_all_finite((_lib.ClipLeaf * 1)(row), -1, P, None), "bad leaf table")
    for over, text, code in (({"grad": None}, "null buffer", 1), ({"size": -1}, "negative size", 1), ({"dtype": 9}, "dtype", 3)):
        bad = _lib.ClipLeaf.from_buffer_copy(row)
        for k, v in over.items():
            setattr(bad, k, v)
        refused(L.rf_all_finite((_lib.ClipLeaf * 1)(bad), 1, P, None), text, code)


def test_the_guard_takes_muon8_and_no_strangers():
    tx = rf.apply_if_finite(rf.muon8(0.1), 1)
    state = tx.init({"w": torch.zeros(4, 8)})
    assert isinstance(state.inner_state, rf.Muon8State)
    with pytest.raises(ValueError, match="ROCm device"):
        tx.update({"w": torch.zeros(4, 8)}, state)
    with pytest.raises(NotImplementedError, match="apply_if_finite wraps"):
        rf.apply_if_finite(rf.clip_by_global_norm(1.0), 1)
