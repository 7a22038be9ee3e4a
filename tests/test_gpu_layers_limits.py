"""Layer operators where their arguments reach a limit: host threads at once, values near the end of a type's range,
rows of any length, parameters outside the arithmetic's range."""
from __future__ import annotations

import ctypes
import pathlib
import subprocess

import numpy as np
import pytest

import layer_reference as ref
from geometricelementaryoperators_b200 import abi
from gpu_helpers import stream, torch
from test_gpu_layers import (EPS, INVALID, P, call, drop_config, like, make, norm_config, parameters, rotary_case,
                             rotary_shape, stats_like, workspace)

pytestmark = pytest.mark.gpu

ROOT = pathlib.Path(__file__).resolve().parent.parent


class LayerLoop(ctypes.Structure):
    """layer_loop_t of c/layer_threads.c."""

    _fields_ = ([(name, ctypes.c_void_p) for name in (
        "norm", "dropout", "x", "weight", "bias", "y", "mean", "rstd", "y_bar", "z_bar", "residual_bar", "x_bar",
        "weight_bar", "bias_bar", "workspace")]
        + [("workspace_bytes", ctypes.c_size_t), ("stream", ctypes.c_void_p), ("calls", ctypes.c_int),
           ("refused", ctypes.c_int)])


@pytest.fixture(scope="module")
def layer_loops(tmp_path_factory):
    out, lib_dir = tmp_path_factory.mktemp("threads") / "layer_threads.so", str(abi.library_path().parent)
    res = subprocess.run(["gcc", "-std=c11", "-O2", "-Wall", "-Wextra", "-shared", "-fPIC", "-pthread", "-I",
                          str(ROOT / "include"), "-I", "/usr/local/cuda/include", str(ROOT / "tests/c/layer_threads.c"),
                          "-o", str(out), "-L", lib_dir, "-lgeo_b200", f"-Wl,-rpath,{lib_dir}"],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    return ctypes.CDLL(str(out)).layer_loops


@pytest.mark.parametrize("kind,widths", [("f32", (4096, 3584)), ("bf16", (4096, 2560)), ("bf16", (16384, 10240))])
def test_two_host_threads_of_unlike_widths(kind, widths, layer_loops):
    """Two host threads, each with a stream, a width and a workspace of its own, call forward and VJP at once: every call
    is taken and gives the bits of one made alone."""
    t = torch()
    dtype = ref.torch_type(kind)
    loops, outs, kept = [], [], []
    for k, cols in enumerate(widths):
        x, dy, dz = (make(40, cols, dtype, seed=10 * k + s) for s in range(3))
        w, b = parameters(cols, dtype)
        n, d = norm_config(x, dtype), drop_config(x, 0.0)
        space, size = workspace(n)
        mean, rstd = stats_like(x)
        y, dx, dres = (t.empty_like(x) for _ in range(3))
        dw, db = t.empty_like(w), t.empty_like(b)
        side = t.cuda.Stream()
        arrays = [P(v) for v in (x, w, b, y, mean, rstd, dy, dz, dres, dx, dw, db, space)]
        loops.append(LayerLoop(ctypes.addressof(n), ctypes.addressof(d), *arrays, size, side.cuda_stream, 4000, 0))
        outs.append((y, mean, rstd, dx, dres, dw, db))
        kept.append((x, dy, dz, w, b, n, d, space, side))
    t.cuda.synchronize()
    alone = []
    for loop, out in zip(loops, outs):
        one = LayerLoop.from_buffer_copy(loop)
        one.calls = 2  # the last call has the cotangent of z, as the last of the loop
        none = LayerLoop.from_buffer_copy(loop)
        none.calls = 0
        assert layer_loops(ctypes.byref(one), ctypes.byref(none)) == 0 and one.refused == 0
        t.cuda.synchronize()
        alone.append([v.clone() for v in out])
    assert layer_loops(ctypes.byref(loops[0]), ctypes.byref(loops[1])) == 0
    t.cuda.synchronize()
    assert [loop.refused for loop in loops] == [0, 0]
    for out, want in zip(outs, alone):
        assert all(t.equal(o, v) for o, v in zip(out, want))


