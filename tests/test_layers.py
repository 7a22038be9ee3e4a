"""Layer operators, the part that needs no GPU: the draws' definition, rotary plans, struct layouts, refusals."""
from __future__ import annotations

import ctypes
import math
import pathlib
import subprocess

import numpy as np
import pytest

import layer_reference as ref
from geometricelementaryoperators_b200 import abi

ROOT = pathlib.Path(__file__).resolve().parent.parent
INVALID = 1
SOME = ctypes.c_void_p(1 << 20)  # never dereferenced: every call here is refused before its arrays are looked at


def test_draws_match_published_vectors():
    """The known answers that come with the generator's paper: all counter and key bits 0, and all 1."""
    assert [int(w) for w in ref.philox(0, 0, 0)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 64) - 1
    assert [int(w) for w in ref.philox(ones, ones, ones)] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_struct_layouts(tmp_path):
    names = {"geo_b200_layer_norm_config_t": abi.LayerNormConfig, "geo_b200_dropout_config_t": abi.DropoutConfig,
             "geo_b200_rotary_config_t": abi.RotaryConfig, "geo_b200_rotary_plan_t": abi.RotaryPlan,
             "geo_b200_rotary_shape_t": abi.RotaryShape}
    lines = []
    for c, py in names.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "geo/geo_b200.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-I", str(ROOT / "include"), "-I",
                    "/usr/local/cuda/include", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in names.values():
        want.append(ctypes.sizeof(py))
        want += [getattr(py, f[0]).offset for f in py._fields_]
    assert got == want


def rotary_config(**k):
    d = dict(layout=abi.ROTARY_HALF, rotary_dim=64, base=10000.0, scaling=abi.ROTARY_SCALING_NONE, factor=4.0,
             original_length=4096.0, low_rotations=1.0, high_rotations=32.0, amplitude=1.0)
    d.update(k)
    return abi.RotaryConfig(**d)


def plan_of(config):
    plan = abi.RotaryPlan()
    return abi.lib().geo_b200_rotary_plan_init(ctypes.byref(plan), ctypes.byref(config)), plan


@pytest.mark.parametrize("dim", [2, 4, 30, 64, 128, 256])
@pytest.mark.parametrize("scaling", ["none", "linear", "base", "banded"])
def test_rotary_plan(dim, scaling):
    """turns + turns_low is the frequency to 2^-62 relative (three extended-precision roundings and the power)."""
    code = ["none", "linear", "base", "banded"].index(scaling)
    status, plan = plan_of(rotary_config(rotary_dim=dim, scaling=code, amplitude=1.25))
    assert status == 0 and plan.rotary_dim == dim and plan.amplitude == 1.25 and plan.layout == abi.ROTARY_HALF
    want = ref.rotary_turns(dim, 10000.0, scaling, 4.0, 4096.0, 1.0, 32.0)
    for i in range(dim // 2):
        got = np.longdouble(plan.turns[i]) + np.longdouble(plan.turns_low[i])
        assert abs(got - want[i]) <= want[i] * 2.0 ** -60
        assert abs(plan.turns_low[i]) <= abs(plan.turns[i]) * 2.0 ** -53
    assert all(plan.turns[i] == 0 for i in range(dim // 2, 128))


def test_rotary_banded_ends():
    """Pairs that turn often over the original context keep their frequency, those that turn rarely are slowed."""
    _, plain = plan_of(rotary_config())
    _, banded = plan_of(rotary_config(scaling=abi.ROTARY_SCALING_BANDED))
    turns = [4096.0 * plain.turns[i] for i in range(32)]
    for i, r in enumerate(turns):
        if r >= 32:
            assert banded.turns[i] == plain.turns[i]
        if r <= 1:
            assert math.isclose(banded.turns[i], plain.turns[i] / 4, rel_tol=1e-15)


@pytest.mark.parametrize("bad", [
    dict(layout=2), dict(rotary_dim=0), dict(rotary_dim=3), dict(rotary_dim=258), dict(base=0.0), dict(base=-1.0),
    dict(base=math.inf), dict(base=math.nan), dict(scaling=4), dict(scaling=1, factor=0.0),
    dict(scaling=1, factor=math.nan), dict(scaling=3, original_length=0.0), dict(scaling=3, low_rotations=32.0),
    dict(scaling=3, high_rotations=math.inf), dict(amplitude=math.nan), dict(amplitude=math.inf),
    dict(base=1e-300),
])
def test_rotary_plan_refusals(bad):
    status, plan = plan_of(rotary_config(**bad))
    assert status == INVALID and plan.rotary_dim == 0  # the plan is left as it was
    L = abi.lib()
    assert L.geo_b200_rotary_plan_init(None, ctypes.byref(rotary_config())) == INVALID
    assert L.geo_b200_rotary_plan_init(ctypes.byref(abi.RotaryPlan()), None) == INVALID


def norm_config(**k):
    d = dict(type=abi.F32, parameter_type=abi.F32, rows=8, cols=64, epsilon=1e-5)
    d.update(k)
    return abi.LayerNormConfig(**d)


BAD_NORM = [dict(type=0), dict(type=5), dict(parameter_type=0), dict(parameter_type=abi.F64),
            dict(type=abi.F64, parameter_type=abi.F32), dict(type=abi.BF16, parameter_type=abi.F16),
            dict(rows=0), dict(cols=0), dict(cols=(1 << 24) + 1), dict(rows=(1 << 32) + 1),
            dict(epsilon=-1e-5), dict(epsilon=math.nan), dict(epsilon=math.inf)]
BAD_STRIDE = [dict(x_stride=63), dict(x_stride=1 << 60)]


@pytest.mark.parametrize("bad", BAD_NORM + BAD_STRIDE)
def test_layer_norm_refusals(bad):
    c = norm_config(**bad)
    L = abi.lib()
    assert L.geo_b200_layer_norm(ctypes.byref(c), SOME, None, None, SOME, None, None, None) == INVALID
    assert L.geo_b200_layer_norm_vjp(ctypes.byref(c), SOME, None, SOME, SOME, SOME, SOME, SOME, SOME, SOME, 1 << 30,
                                     None) == INVALID
    if "x_stride" not in bad:
        assert L.geo_b200_layer_norm_vjp_workspace(ctypes.byref(c)) == 0


def test_layer_norm_null_arguments():
    c, L = norm_config(), abi.lib()
    r = ctypes.byref(c)
    assert L.geo_b200_layer_norm(None, SOME, None, None, SOME, None, None, None) == INVALID
    assert L.geo_b200_layer_norm(r, None, None, None, SOME, None, None, None) == INVALID
    assert L.geo_b200_layer_norm(r, SOME, None, None, None, None, None, None) == INVALID
    full = [r, SOME, None, SOME, SOME, SOME, SOME, SOME, SOME, SOME, 1 << 30, None]
    for missing in (0, 1, 3, 4, 5):
        args = list(full)
        args[missing] = None
        assert L.geo_b200_layer_norm_vjp(*args) == INVALID
    args = list(full)
    args[6] = args[7] = args[8] = None  # no output at all
    assert L.geo_b200_layer_norm_vjp(*args) == INVALID
    assert L.geo_b200_layer_norm_vjp_workspace(None) == 0
    assert L.geo_b200_layer_norm_vjp_workspace(r) >= 2 * 64 * 4
    # In place needs the same stride on both sides.
    c2 = norm_config(x_stride=64, y_stride=72)
    assert L.geo_b200_layer_norm(ctypes.byref(c2), SOME, None, None, SOME, None, None, None) == INVALID


def drop_config(**k):
    d = dict(type=abi.F32, dimension=0, rows=8, cols=64, rate=0.1, seed=1, offset=2)
    d.update(k)
    return abi.DropoutConfig(**d)


@pytest.mark.parametrize("bad", [
    dict(type=0), dict(type=9), dict(dimension=7), dict(cols=66, dimension=2), dict(rows=0), dict(cols=0),
    dict(rate=-0.1), dict(rate=1.5), dict(rate=math.nan), dict(x_stride=8, y_cotangent_stride=8),
    dict(y_stride=63, x_cotangent_stride=63), dict(cols=(1 << 24) + 64)])
def test_dropout_refusals(bad):
    c, n, L = drop_config(**bad), norm_config(), abi.lib()
    assert L.geo_b200_dropout(ctypes.byref(c), SOME, None, None, SOME, None) == INVALID
    assert L.geo_b200_dropout_vjp(ctypes.byref(c), None, SOME, SOME, None) == INVALID
    assert L.geo_b200_residual_dropout_layer_norm(ctypes.byref(n), ctypes.byref(c), SOME, SOME, None, None, None,
                                                  SOME, ctypes.c_void_p(1 << 24), None, None, None) == INVALID


def test_dropout_null_arguments():
    r, L = ctypes.byref(drop_config()), abi.lib()
    assert L.geo_b200_dropout(None, SOME, None, None, SOME, None) == INVALID
    assert L.geo_b200_dropout(r, None, None, None, SOME, None) == INVALID
    assert L.geo_b200_dropout(r, SOME, None, None, None, None) == INVALID
    assert L.geo_b200_dropout_vjp(None, None, SOME, SOME, None) == INVALID
    assert L.geo_b200_dropout_vjp(r, None, None, SOME, None) == INVALID
    assert L.geo_b200_dropout_vjp(r, None, SOME, None, None) == INVALID


@pytest.mark.parametrize("n,d", [
    (dict(type=abi.BF16), dict()), (dict(rows=9), dict()), (dict(cols=128), dict()), (dict(x_stride=72), dict()),
    (dict(), dict(y_stride=72)), (dict(epsilon=-1.0), dict())])
def test_fused_refusals(n, d):
    """The two configs have to agree on type, rows, cols and z's stride."""
    n, d, L = norm_config(**n), drop_config(**d), abi.lib()
    a, b = ctypes.byref(n), ctypes.byref(d)
    other = ctypes.c_void_p(1 << 24)
    assert L.geo_b200_residual_dropout_layer_norm(a, b, SOME, SOME, None, None, None, SOME, other, None, None,
                                                  None) == INVALID
    assert L.geo_b200_residual_dropout_layer_norm_vjp(a, b, None, SOME, None, SOME, SOME, SOME, None, SOME, other,
                                                      None, None, None, 0, None) == INVALID


def test_fused_null_arguments():
    n, d, L = norm_config(), drop_config(), abi.lib()
    a, b, other = ctypes.byref(n), ctypes.byref(d), ctypes.c_void_p(1 << 24)
    forward = [a, b, SOME, SOME, None, None, None, SOME, other, None, None, None]
    for missing in (0, 1, 2, 3, 7, 8):
        args = list(forward)
        args[missing] = None
        assert L.geo_b200_residual_dropout_layer_norm(*args) == INVALID
    args = list(forward)
    args[8] = SOME  # y and z in one array
    assert L.geo_b200_residual_dropout_layer_norm(*args) == INVALID
    backward = [a, b, None, SOME, None, SOME, SOME, SOME, None, SOME, other, None, None, None, 0, None]
    for missing in (0, 1, 3, 5, 6, 7):
        args = list(backward)
        args[missing] = None
        assert L.geo_b200_residual_dropout_layer_norm_vjp(*args) == INVALID
    args = list(backward)
    args[9] = args[10] = None
    assert L.geo_b200_residual_dropout_layer_norm_vjp(*args) == INVALID
    args = list(backward)
    args[10] = SOME  # both outputs in one array
    assert L.geo_b200_residual_dropout_layer_norm_vjp(*args) == INVALID


def rotary_shape(**k):
    d = dict(type=abi.F32, position_type=abi.I64, batch=2, tokens=3, heads=4, head_dim=64)
    d.update(k)
    return abi.RotaryShape(**d)


@pytest.mark.parametrize("bad", [
    dict(type=0), dict(type=5), dict(position_type=0), dict(position_type=3), dict(batch=0), dict(tokens=0),
    dict(heads=0), dict(head_dim=63), dict(head_dim=65537), dict(y_head_stride=63), dict(y_token_stride=255),
    dict(y_batch_stride=767), dict(x_batch_stride=1 << 60), dict(tokens=1 << 62), dict(heads=1 << 62),
    dict(first_position=(1 << 31) - 1), dict(first_position=-(1 << 31) - 1), dict(tokens=(1 << 31) + 5, batch=1)])
def test_rotary_refusals(bad):
    _, plan = plan_of(rotary_config())
    s, L = rotary_shape(**bad), abi.lib()
    other = ctypes.c_void_p(1 << 24)
    for call in (L.geo_b200_rotary, L.geo_b200_rotary_vjp):
        assert call(ctypes.byref(plan), ctypes.byref(s), SOME, None, other, None) == INVALID


def test_rotary_null_and_bad_plans():
    _, plan = plan_of(rotary_config())
    s, L = rotary_shape(), abi.lib()
    p, q = ctypes.byref(plan), ctypes.byref(s)
    for call in (L.geo_b200_rotary, L.geo_b200_rotary_vjp):
        assert call(None, q, SOME, None, SOME, None) == INVALID
        assert call(p, None, SOME, None, SOME, None) == INVALID
        assert call(p, q, None, None, SOME, None) == INVALID
        assert call(p, q, SOME, None, None, None) == INVALID
        assert call(ctypes.byref(abi.RotaryPlan()), q, SOME, None, SOME, None) == INVALID  # never initialised
        moved = rotary_shape(x_head_stride=64, y_head_stride=72)
        assert call(p, ctypes.byref(moved), SOME, None, SOME, None) == INVALID  # in place, another stride


@pytest.mark.parametrize("name", ["x_stride", "y_cotangent_stride", "x_cotangent_stride"])
@pytest.mark.parametrize("stride", [63, 1 << 60])
def test_vjp_workspace_of_refused_strides(name, stride):
    """0 bytes for whatever the VJP refuses, its strides among it; the forward's own stride does not matter."""
    L = abi.lib()
    c = norm_config(**{name: stride})
    assert L.geo_b200_layer_norm_vjp(ctypes.byref(c), SOME, None, SOME, SOME, SOME, SOME, SOME, SOME, SOME, 1 << 30,
                                     None) == INVALID
    assert L.geo_b200_layer_norm_vjp_workspace(ctypes.byref(c)) == 0
    packed = L.geo_b200_layer_norm_vjp_workspace(ctypes.byref(norm_config()))
    assert packed > 0
    assert L.geo_b200_layer_norm_vjp_workspace(ctypes.byref(norm_config(**{name: 72}))) == packed
    assert L.geo_b200_layer_norm_vjp_workspace(ctypes.byref(norm_config(y_stride=stride))) == packed
