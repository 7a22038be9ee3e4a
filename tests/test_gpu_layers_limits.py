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
from test_gpu_layers import (EPS, INVALID, KINDS, P, call, drop_bound, drop_config, like, make, mask, norm_config,
                             parameters, rotary_case, rotary_shape, stats_like, untouched, workspace)
from test_gpu_layers import test_layer_norm as check_layer_norm
from test_gpu_layers import test_layer_norm_in_place_and_without_parameters as check_in_place
from test_gpu_layers import test_layer_norm_non_finite_rows_stay_apart as check_non_finite
from test_gpu_layers import test_layer_norm_vjp as check_layer_norm_vjp
from test_gpu_layers import test_residual_dropout_layer_norm as check_fused
from test_gpu_layers import test_residual_dropout_layer_norm_vjp as check_fused_vjp

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


#: Additions along the longest path of a row's or a column's sum in the kernels for rows of any length: 64 values one
#: after another in a thread, 64 of those sums, the rest (cols / 2^20, rows / 2^15), a warp's 5 steps, 8 warps or groups,
#: and 3 for the division and the result.
LONG_PATH = 64 + 64 + 16 + 5 + 8 + 3


@pytest.mark.parametrize("cols", [(1 << 20) + 3, 1 << 22, 1 << 24])
@pytest.mark.parametrize("value", [0.1, 1.1])
def test_statistics_of_long_rows_of_one_value(cols, value):
    """Equal values round the same way at every addition: the error of a long chain of them grows with its length, that
    of sums of sums does not."""
    t = torch()
    x = t.full((2, cols), value, device="cuda")
    zero = t.zeros_like(x)
    y, z = t.empty_like(x), t.empty_like(x)
    mean, rstd = stats_like(x)
    n, d = norm_config(x, t.float32), drop_config(x, 0.0)
    want = [torch().tensor(v, device="cuda", dtype=t.float64) for v in (0.0, float(x[0, 0]), EPS ** -0.5)]
    bounds = [float(v.max()) for v in ref.norm_bound(x[:, :8].double(), None, None, want[2].expand(2), want[0], t.float32,
                                                     LONG_PATH)]
    for fused in (False, True):
        if fused:
            call("geo_b200_residual_dropout_layer_norm", ctypes.byref(n), ctypes.byref(d), P(x), P(zero), None, None, None,
                 P(z), P(y), P(mean), P(rstd))
            assert t.equal(z, x)
        else:
            call("geo_b200_layer_norm", ctypes.byref(n), P(x), None, None, P(y), P(mean), P(rstd))
        for got, v, bound, what in zip((y, mean, rstd), want, bounds, ("y", "mean", "rstd")):
            assert float((got.double() - v).abs().max()) <= bound, (what, fused)


@pytest.mark.parametrize("value", [0.1, 1.1])
def test_vjp_of_long_rows_of_one_cotangent(value):
    t = torch()
    cols = 1 << 22
    x = make(2, cols, t.float32, seed=3)
    dy = t.full_like(x, value)
    _, mean, rstd = ref.norm(x.double(), None, None, EPS)
    mean, rstd = mean.float(), rstd.float()
    dx = t.empty_like(x)
    call("geo_b200_layer_norm_vjp", ctypes.byref(norm_config(x, t.float32)), P(x), None, P(mean), P(rstd), P(dy), P(dx),
         None, None, None, 0)
    wide = [x.double(), None, mean.double(), rstd.double(), dy.double()]
    want = ref.norm_vjp(*wide)[0]
    ref.assert_within(dx, want, ref.norm_vjp_bound(*wide, want, t.float32, LONG_PATH)[0], "dx")


@pytest.mark.parametrize("value", [0.1, 1.1])
def test_column_sums_over_many_long_rows(value):
    """32776 columns, 32768 rows of one cotangent: bias_bar is rows times it."""
    t = torch()
    rows, cols = 1 << 15, 32776
    x = t.zeros(rows, cols, device="cuda")
    dy = t.full_like(x, value)
    mean, rstd = t.full((rows,), -1.0, device="cuda"), t.full((rows,), 1.0, device="cuda")
    n = norm_config(x, t.float32)
    space, size = workspace(n)
    dw, db = (t.empty(cols, device="cuda") for _ in range(2))
    call("geo_b200_layer_norm_vjp", ctypes.byref(n), P(x), None, P(mean), P(rstd), P(dy), None, P(dw), P(db), P(space), size)
    want = rows * float(dy[0, 0])
    for got in (dw, db):  # xh = 1: the same sum
        assert float((got.double() - want).abs().max()) <= LONG_PATH * 2.0 ** -24 * want


@pytest.mark.parametrize("cols", [8192, 16384, 32768])
@pytest.mark.parametrize("backward", [False, True])
def test_wait_of_a_cluster_that_gives_up(cols, backward):
    """A block that sends nothing in one round: rows before it are right; that one and all later ones, their statistics
    and the column sums are NaN; the context stays usable. A round that does not come changes nothing."""
    t = torch()
    L = abi.lib()
    rows = 1200
    x, dy = make(rows, cols, t.float32, seed=1, shift=0.5), make(rows, cols, t.float32, seed=2)
    _, m, r = ref.norm(x.double(), None, None, EPS)
    n = norm_config(x, t.float32, x_stride=0, y_stride=0, y_cotangent_stride=0, x_cotangent_stride=0)
    space, size = workspace(n)
    out, want = t.full_like(x, 7.0), t.empty_like(x)
    stats = [m.float(), r.float()] if backward else stats_like(x)
    sums = [t.full((cols,), 7.0, device="cuda") for _ in range(2)]

    def usual():
        """The ordinary call's results."""
        s, v = [p.clone() for p in stats], [t.empty_like(p) for p in sums]
        if backward:
            call("geo_b200_layer_norm_vjp", ctypes.byref(n), P(x), None, P(s[0]), P(s[1]), P(dy), P(want), P(v[0]), P(v[1]),
                 P(space), size)
        else:
            call("geo_b200_layer_norm", ctypes.byref(n), P(x), None, None, P(want), P(s[0]), P(s[1]))
        return [want] + (v if backward else s)

    def starved(round, polls):
        call("geo_b200_layer_norm_wait_selftest", ctypes.byref(n), P(x), P(dy) if backward else None, P(out), P(stats[0]),
             P(stats[1]), P(sums[0]), P(sums[1]), P(space), size, round, polls)
        t.cuda.synchronize()
        return [out] + (sums if backward else stats)

    for round in (1, 2):
        clean = [v.clone() for v in usual()]
        got = starved(round, 1 << 14)
        bad = t.isnan(out).any(1)
        first = int(bad.int().argmax())
        assert 0 < first <= rows // 2 and first % round == 0
        assert t.isnan(out[first:]).all() and t.equal(out[:first], clean[0][:first])
        for v, w in zip(got[1:], clean[1:]):
            if backward:
                assert t.isnan(v).all()
            else:
                assert t.isnan(v[first:]).all() and t.equal(v[:first], w[:first])
        again = usual()
        assert all(t.equal(v, w) for v, w in zip(again, clean))
    assert all(t.equal(v, w) for v, w in zip(starved(1 << 20, 1 << 14), clean))
    refused = [dict(type=abi.F64, parameter_type=abi.F64), dict(cols=4096), dict(cols=cols - 4), dict(x_stride=cols),
               dict(epsilon=-1.0)]
    for bad in refused:
        c = norm_config(x, t.float32, **{**dict(x_stride=0, y_stride=0, y_cotangent_stride=0, x_cotangent_stride=0), **bad})
        assert L.geo_b200_layer_norm_wait_selftest(ctypes.byref(c), P(x), None, P(out), P(stats[0]), P(stats[1]), None, None,
                                                   None, 0, 1, 64, stream()) == INVALID
    assert L.geo_b200_layer_norm_wait_selftest(ctypes.byref(n), P(x), None, P(out), P(stats[0]), P(stats[1]), None, None,
                                               None, 0, 1, 0, stream()) == INVALID


# Rows beyond the clusters' length (32768 values, 16384 in float64), for every type: packed, many, off 16 bytes.
@pytest.mark.parametrize("kind,pkind", KINDS)
@pytest.mark.parametrize("rows,cols,pad", [(3, 32769, 0), (70, 40000, 0), (2, 100003, 1), (200, 33000, 8)])
def test_layer_norm_of_rows_of_any_length(kind, pkind, rows, cols, pad):
    check_layer_norm(kind, pkind, rows, cols, pad)
    check_layer_norm_vjp(kind, pkind, rows, cols, pad)


@pytest.mark.parametrize("kind,pkind", KINDS)
@pytest.mark.parametrize("rows,cols,pad,dimension", [(3, 32769, 0, 0), (70, 40000, 0, 6), (2, 100003, 1, 0), (200, 33000, 8, 3)])
def test_residual_dropout_layer_norm_of_rows_of_any_length(kind, pkind, rows, cols, pad, dimension):
    check_fused(kind, pkind, rows, cols, pad, dimension)
    check_fused_vjp(kind, pkind, rows, cols, pad, dimension)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols,pad", [(32776, 0), (40001, 1)])
def test_rows_of_any_length_in_place_and_non_finite(kind, cols, pad):
    check_in_place(kind, cols, pad)
    check_non_finite(kind, cols)


@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,pads", [(50, 100, (1, 0, 3, 2)), (9, 1003, (0, 5, 1, 2)), (7, 5001, (2, 3, 0, 1)),
                                            (130, 13, (0, 1, 2, 3)), (3, 33001, (1, 2, 0, 3))])
def test_dropped_cotangent_of_arrays_of_unlike_alignment(kind, rows, cols, pads):
    """x_bar of the fused VJP, every array with a stride and an alignment of its own: kept values scaled, dropped ones 0."""
    t = torch()
    dtype = ref.torch_type(kind)
    z, dy, dz, other = (make(rows, cols, dtype, p, seed=i, shift=0.2) for i, p in enumerate(pads))
    w, b = parameters(cols, dtype)
    _, mean, rstd = ref.norm(z.double(), None, None, EPS)
    mean, rstd = mean.to(ref.wide_type(dtype)), rstd.to(ref.wide_type(dtype))
    (dres, rw), (dx, xw) = like(dy), like(other)
    rate = 0.3
    n = norm_config(z, dtype, y_cotangent_stride=dy.stride(0), x_cotangent_stride=dres.stride(0))
    d = drop_config(z, rate, y_stride=z.stride(0), y_cotangent_stride=dz.stride(0), x_cotangent_stride=dx.stride(0))
    keep = mask(d)
    call("geo_b200_residual_dropout_layer_norm_vjp", ctypes.byref(n), ctypes.byref(d), None, P(z), P(w), P(mean), P(rstd),
         P(dy), P(dz), P(dres), P(dx), None, None, None, 0)
    wide = [v.double() for v in (z, w, mean, rstd, dy)]
    want = ref.norm_vjp(*wide)[0] + dz.double()
    bounds = ref.norm_vjp_bound(*wide, want, dtype, max(ref.PATH, cols // 100))
    inner = bounds[0] - ref.half_step(dtype) * want.abs() + ref.u_wide(dtype) * want.abs()
    ref.assert_within(dres, want, bounds[0] + ref.u_wide(dtype) * want.abs(), "dresidual")
    want_dx = t.where(keep, want * ref.scale(rate), t.zeros_like(want))
    ref.assert_within(dx, want_dx, drop_bound(want, keep, rate, want_dx, dtype) + ref.scale(rate) * inner, "dx")
    assert untouched(rw, cols) and untouched(xw, cols)


@pytest.mark.parametrize("kind", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_at_the_highest_frequencies(kind, layout):
    """A base below 1 makes frequencies up to the largest that a plan takes (2^18 turns a position): at far positions the
    angle's own error, 2^-63 |position| turns times the turns a position, is what the result is off by."""
    t = torch()
    x = rotary_case(kind, 1, 6, 3, 64)
    positions = np.array([[-(1 << 31), (1 << 31) - 1, 1 << 31, 1234567891, -2147483647, 77]])
    c = abi.RotaryConfig(layout=abi.ROTARY_HALF if layout == "half" else abi.ROTARY_INTERLEAVED, rotary_dim=64, base=4e-7,
                         scaling=abi.ROTARY_SCALING_NONE, amplitude=1.0)
    plan = abi.RotaryPlan()
    assert abi.lib().geo_b200_rotary_plan_init(ctypes.byref(plan), ctypes.byref(c)) == 0
    turns = ref.rotary_turns(64, 4e-7)
    assert 2 ** 17 < turns[-1] <= 2 ** 18
    for name, backward in (("geo_b200_rotary", False), ("geo_b200_rotary_vjp", True)):
        y = t.empty_like(x)
        call(name, ctypes.byref(plan), ctypes.byref(rotary_shape(x, y, position_batch_stride=6)), P(x),
             P(t.tensor(positions, device="cuda")), P(y))
        want = ref.rotary(x.double(), positions, turns, layout, 1.0, backward)
        ref.assert_within(y, want, ref.rotary_bound(x.double(), want, turns, layout, 1.0, x.dtype, 1 << 31), name)


@pytest.mark.parametrize("kind,cols", [("f32", 8192), ("bf16", 5120), ("bf16", 4096), ("f16", 8001), ("f32", 33000)])
def test_captured_graph_of_wide_rows(kind, cols):
    """Forward and VJP of rows in blocks, in clusters and of any length, captured and replayed on other inputs: the bits
    of eager calls, while eager calls with a workspace of their own run on another stream."""
    t = torch()
    dtype = ref.torch_type(kind)
    x, res, dy, dz = (make(300, cols, dtype, seed=s) for s in range(4))
    w, b = parameters(cols, dtype)
    n, d = norm_config(x, dtype), drop_config(x, 0.4)
    outs, spaces = [], []
    for _ in range(2):
        outs.append([t.empty_like(x) for _ in range(4)] + stats_like(x) + [t.empty_like(w), t.empty_like(b)])
        spaces.append(workspace(n))

    def step(k):
        z, y, dres, dx, mean, rstd, dw, db = outs[k]
        call("geo_b200_residual_dropout_layer_norm", ctypes.byref(n), ctypes.byref(d), P(x), P(res), None, P(w), P(b), P(z),
             P(y), P(mean), P(rstd))
        call("geo_b200_residual_dropout_layer_norm_vjp", ctypes.byref(n), ctypes.byref(d), None, P(z), P(w), P(mean),
             P(rstd), P(dy), P(dz), P(dres), P(dx), P(dw), P(db), P(spaces[k][0]), spaces[k][1])

    side, graph = t.cuda.Stream(), t.cuda.CUDAGraph()
    side.wait_stream(t.cuda.current_stream())
    with t.cuda.graph(graph, stream=side):
        step(0)
    for s in range(3):
        for k, v in enumerate((x, res, dy, dz)):
            v.copy_(make(300, cols, dtype, seed=100 + 10 * s + k))
        t.cuda.synchronize()
        for _ in range(3):
            with t.cuda.stream(side):
                graph.replay()
            step(1)
        t.cuda.synchronize()
        assert all(t.equal(p, q) for p, q in zip(*outs))


def test_wait_selftest_refuses_longer_waits():
    t = torch()
    x = make(4, 8192, t.float32)
    y, _ = like(x)
    mean, rstd = stats_like(x)
    n = norm_config(x, t.float32, x_stride=0, y_stride=0, y_cotangent_stride=0, x_cotangent_stride=0)
    for polls, status in ((1 << 22, 0), ((1 << 22) + 1, INVALID), ((1 << 32) - 1, INVALID)):
        assert abi.lib().geo_b200_layer_norm_wait_selftest(ctypes.byref(n), P(x), None, P(y), P(mean), P(rstd), None, None,
                                                           None, 0, 1000, polls, stream()) == status  # no such round
