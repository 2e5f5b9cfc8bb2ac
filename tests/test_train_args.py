"""The training-step entries refuse bad arguments before any CUDA call: no GPU
needed, the pointers are never dereferenced."""
from __future__ import annotations

import ctypes
import math
from array import array

import pytest

from conftest import spmd_mod

P = 0x100000  # a plausible, aligned address


def lib():
    return spmd_mod("_lib").lib()


def ptr(a):
    return a.buffer_info()[0] if a is not None else None


def norm_args(**kw):
    a = {"rank": 2, "sizes": [4, 32], "x": P, "xt": 0, "xs": [32, 1], "y": 2 * P, "yt": 0, "ys": [32, 1], "w": 3 * P,
         "b": 4 * P, "wt": 0, "eps": 1e-5, "mean": 5 * P, "rstd": 6 * P, "ws": None, "bytes": 0}
    a.update(kw)
    arrays = [array("q", a[n]) if a[n] is not None else None for n in ("sizes", "xs", "ys")]
    st = lib().spmdb200_layer_norm(a["rank"], ptr(arrays[0]), a["x"], a["xt"], ptr(arrays[1]), a["y"], a["yt"],
                                   ptr(arrays[2]), a["w"], a["b"], a["wt"], a["eps"], a["mean"], a["rstd"], a["ws"],
                                   a["bytes"], None)
    return st


@pytest.mark.parametrize("bad", [
    {"rank": 0}, {"rank": 4}, {"sizes": None}, {"sizes": [4, 0]}, {"sizes": [-1, 32]}, {"sizes": [1 << 41, 32]},
    {"x": None}, {"y": None}, {"xs": None}, {"ys": None}, {"x": P + 2}, {"y": 2 * P + 1}, {"w": 3 * P + 2},
    {"mean": 5 * P + 1}, {"xt": 3}, {"yt": -1}, {"wt": 7}, {"eps": -1.0}, {"eps": math.nan}, {"xs": [32, -1]},
    {"ys": [0, 1]}, {"ys": [31, 1]}, {"ys": [32, 0]}, {"ys": [1, 1]}, {"ys": [2, 5]},
])
def test_layer_norm_refuses(bad):
    assert norm_args(**bad) == -1
    assert lib().spmdb200_last_error_message()


def test_layer_norm_refuses_type_pairs_and_many_rows():
    assert norm_args(xt=1, yt=2) == -4
    assert norm_args(rank=3, sizes=[1 << 30, 1 << 30, 4], xs=[4, 4, 1], ys=[1 << 32, 4, 1]) == -1
    long = {"sizes": [4, 60000], "xs": [60000, 1], "ys": [60000, 1]}  # rows that need a workspace
    assert norm_args(**long) == -5 and norm_args(**long, ws=7 * P + 8, bytes=1 << 30) == -5
    assert norm_args(**long, ws=7 * P, bytes=64) == -5


def test_layer_norm_accepts():
    """No rows needs no pointer; strides of a size-1 dimension do not matter; column-major output is no overlap."""
    assert norm_args(sizes=[0, 32], x=None, y=None) == 0
    import torch
    if torch.cuda.is_available():
        return  # what follows would launch
    assert norm_args(sizes=[1, 32], ys=[0, 1]) == -6
    assert norm_args(ys=[1, 4]) == -6
    assert norm_args(rank=3, sizes=[2, 3, 8], xs=[0, 0, 0], ys=[8, 16, 1]) == -6


def back_args(**kw):
    a = {"sizes": [4, 32], "dy": P, "gt": 0, "gs": [32, 1], "x": 2 * P, "xt": 0, "xs": [32, 1], "mean": 3 * P,
         "rstd": 4 * P, "w": 5 * P, "wt": 0, "dx": 6 * P, "ds": [32, 1], "dw": 7 * P, "db": 8 * P, "dt": 0, "ws": 9 * P,
         "bytes": 1 << 20}
    a.update(kw)
    s, gs, xs, ds = (array("q", a[n]) if a[n] is not None else None for n in ("sizes", "gs", "xs", "ds"))
    return lib().spmdb200_layer_norm_backward(2, ptr(s), a["dy"], a["gt"], ptr(gs), a["x"], a["xt"], ptr(xs), a["mean"],
                                              a["rstd"], a["w"], a["wt"], a["dx"], ptr(ds), a["dw"], a["db"], a["dt"],
                                              a["ws"], a["bytes"], None)


@pytest.mark.parametrize("bad,status", [
    ({"dy": None}, -1), ({"x": None}, -1), ({"mean": None}, -1), ({"rstd": None}, -1), ({"ds": None}, -1),
    ({"ds": [16, 1]}, -1), ({"gt": 5}, -1), ({"wt": 5}, -1), ({"dt": 5}, -1), ({"xt": 1, "gt": 2}, -4),
    ({"dx": 6 * P + 1}, -1), ({"dw": 7 * P + 1}, -1), ({"ws": None}, -5), ({"ws": 9 * P + 8}, -5), ({"bytes": 8}, -5),
])
def test_layer_norm_backward_refuses(bad, status):
    assert back_args(**bad) == status


def test_workspace_sizes():
    f = lib().spmdb200_layer_norm_workspace_bytes
    assert f(-1, 4) == 0 and f(4, 0) == 0
    for rows in (0, 1, 100, 1 << 20):
        for cols in (1, 64, 1000, 8192, 8193, 100000, 1 << 18, 1 << 24):
            # Column sums of at most 444 rows of 8192 or so, or eight partial rows; shares of 72 MB of rows, or of eight.
            assert 8 * cols <= f(rows, cols) <= (32 << 20) + 80 * cols, (rows, cols)
            assert lib().spmdb200_layer_norm_forward_workspace_bytes(rows, cols) <= (8 << 20) + 2 * cols, (rows, cols)
    for cols in (8185, 20000, 49145):
        assert lib().spmdb200_layer_norm_forward_workspace_bytes(1000, cols) == 0
    assert lib().spmdb200_layer_norm_forward_workspace_bytes(1000, 49146) > 0
    g = lib().spmdb200_grad_norm_workspace_bytes
    assert 0 < g(0) <= g(1) <= g(5000) <= 1 << 20


def adam_args(n=2, **kw):
    a = {"params": [P, 2 * P], "pt": [0, 0], "grads": [3 * P, 4 * P], "gt": [2, 2], "sizes": [100, 200],
         "m": [5 * P, 6 * P], "v": [7 * P, 8 * P], "bits": 32, "ms": None, "vs": None, "copies": None, "ct": None,
         "decay": [0.0, 0.1], "lr": 1e-3, "lr_dev": None, "b1": 0.9, "b2": 0.99, "eps": 1e-8, "step": 1,
         "step_dev": None, "scale": None}
    a.update(kw)
    kinds = {"params": "Q", "grads": "Q", "m": "Q", "v": "Q", "ms": "Q", "vs": "Q", "copies": "Q", "pt": "i", "gt": "i",
             "ct": "i", "sizes": "q", "decay": "d"}
    h = {k: array(t, a[k]) if a[k] is not None else None for k, t in kinds.items()}
    return lib().spmdb200_adamw(n, ptr(h["params"]), ptr(h["pt"]), ptr(h["grads"]), ptr(h["gt"]), ptr(h["sizes"]),
                                ptr(h["m"]), ptr(h["v"]), a["bits"], ptr(h["ms"]), ptr(h["vs"]), ptr(h["copies"]),
                                ptr(h["ct"]), ptr(h["decay"]), a["lr"], a["lr_dev"], a["b1"], a["b2"], a["eps"],
                                a["step"], a["step_dev"], a["scale"], None)


@pytest.mark.parametrize("bad", [
    {"n": -1}, {"params": None}, {"grads": None}, {"m": None}, {"v": None}, {"sizes": None}, {"decay": None},
    {"pt": None}, {"bits": 16}, {"bits": 8}, {"bits": 8, "ms": [9 * P, 10 * P], "vs": [11 * P, 0]},
    {"params": [P, 0]}, {"grads": [0, P]}, {"m": [0, 6 * P]}, {"sizes": [100, -1]}, {"pt": [0, 3]}, {"gt": [-1, 0]},
    {"params": [P + 2, 2 * P]}, {"m": [5 * P + 2, 6 * P]}, {"copies": [9 * P, 0]}, {"copies": [9 * P, 0], "ct": [0, 0]},
    {"copies": [9 * P + 1, 0], "ct": [1, 0]}, {"b1": 1.0}, {"b2": -0.5}, {"b1": math.nan}, {"eps": -1.0}, {"lr": -1.0},
    {"lr": math.nan}, {"step": 0}, {"decay": [0.0, -1.0]}, {"decay": [math.nan, 0.0]}, {"lr_dev": P + 1},
    {"step_dev": P + 4}, {"scale": P + 2},
    # overlaps: twice the same parameter, a state inside a parameter, a gradient that is a parameter, scales that meet
    {"params": [P, P]}, {"params": [P, P + 396]}, {"m": [5 * P, P + 4]}, {"v": [5 * P, 8 * P]}, {"grads": [2 * P, 4 * P]},
    {"copies": [P, 0], "ct": [1, 0]},
    {"bits": 8, "ms": [9 * P, 10 * P], "vs": [9 * P, 11 * P]},
])
def test_adamw_refuses(bad):
    assert adam_args(**bad) == -1
    assert lib().spmdb200_last_error_message()


def test_adamw_accepts():
    """Empty lists and empty tensors do nothing; a gradient may be listed twice."""
    assert adam_args(n=0, params=None, grads=None) == 0
    assert adam_args(sizes=[0, 0], params=[0, 0], grads=[0, 0], m=[0, 0], v=[0, 0]) == 0
    import torch
    if torch.cuda.is_available():
        return  # what follows would launch
    assert adam_args(grads=[3 * P, 3 * P]) == -6
    assert adam_args(params=[P, P + 400]) == -6


def grad_args(n=1, grads=(P,), sizes=(10,), types=(0,), max_norm=1.0, norm=2 * P, scale=3 * P, ws=4 * P, nbytes=1 << 20):
    a = [array(t, v) if v is not None else None for t, v in (("Q", grads), ("q", sizes), ("i", types))]
    return lib().spmdb200_grad_norm(n, ptr(a[0]), ptr(a[1]), ptr(a[2]), max_norm, norm, scale, ws, ctypes.c_size_t(nbytes), None)


@pytest.mark.parametrize("bad,status", [
    ({"n": -1}, -1), ({"grads": None}, -1), ({"sizes": None}, -1), ({"types": None}, -1), ({"grads": (0,)}, -1),
    ({"grads": (P + 2,)}, -1), ({"sizes": (-1,)}, -1), ({"types": (5,)}, -1), ({"norm": None}, -1), ({"norm": P + 1}, -1),
    ({"max_norm": -1.0}, -1), ({"max_norm": math.nan}, -1), ({"ws": None}, -5), ({"ws": 4 * P + 8}, -5), ({"nbytes": 8}, -5),
])
def test_grad_norm_refuses(bad, status):
    assert grad_args(**bad) == status


def test_python_wrappers_refuse_host_tensors():
    import torch
    k = spmd_mod("kernels")
    x, w = torch.ones(4, 8), [torch.ones(8)]
    for call in (lambda: k.layer_norm(x), lambda: k.layer_norm_backward(x, x, x[:, 0], x[:, 0]),
                 lambda: k.grad_norm(w, 1.0), lambda: k.adamw(w, w, w, w, step=1, lr=0.1)):
        with pytest.raises(ValueError):
            call()
