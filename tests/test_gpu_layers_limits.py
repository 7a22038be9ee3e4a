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


@pytest.mark.parametrize("kind", ["bf16", "f32", "f64"])
@pytest.mark.parametrize("cols", [8, 24, 32, 25, 72, 1000, 1024, 1003, 3000, 4096, 5128, 8192, 40000])
@pytest.mark.parametrize("fused", [False, True])
def test_vjp_of_constant_rows_near_the_end_of_the_range(kind, cols, fused):
    """Rows of one value v, whose own (v - mean) rstd is 0 while v rstd overflows: the formula's finite x_bar, at widths
    that fill a team of threads and at those that do not."""
    t = torch()
    dtype = ref.torch_type(kind)
    x, dy, dz = (make(9, cols, dtype, seed=s) for s in range(3))
    w, b = parameters(cols, dtype)
    _, mean, rstd = ref.norm(x.double(), None, None, EPS)
    for row in (0, 4, 8):
        x[row] = 1e306 if kind == "f64" else 2e36
        mean[row], rstd[row] = x[row, 0].double(), EPS ** -0.5
    x[4] *= -1
    mean[4] *= -1
    mean, rstd = mean.to(ref.wide_type(dtype)), rstd.to(ref.wide_type(dtype))
    n, d = norm_config(x, dtype), drop_config(x, 0.0)
    space, size = workspace(n)
    dx = t.empty_like(x)
    dw, db = t.empty_like(w), t.empty_like(b)
    if fused:
        call("geo_b200_residual_dropout_layer_norm_vjp", ctypes.byref(n), ctypes.byref(d), None, P(x), P(w), P(mean),
             P(rstd), P(dy), P(dz), P(dx), None, P(dw), P(db), P(space), size)
    else:
        call("geo_b200_layer_norm_vjp", ctypes.byref(n), P(x), P(w), P(mean), P(rstd), P(dy), P(dx), P(dw), P(db), P(space),
             size)
    wide = [v.double() for v in (x, w, mean, rstd, dy)]
    want = ref.norm_vjp(*wide)
    total = want[0] + dz.double() if fused else want[0]
    bounds = ref.norm_vjp_bound(*wide, total, dtype, max(ref.PATH, cols // 100))
    u = ref.half_step(dtype)
    ref.assert_within(dx, total, bounds[0] + ref.u_wide(dtype) * total.abs(), "dx")
    ref.assert_within(dw, want[1], bounds[1] + u * want[1].abs() + ref.least(dtype), "dweight")
    ref.assert_within(db, want[2], bounds[2] + u * want[2].abs() + ref.least(dtype), "dbias")


