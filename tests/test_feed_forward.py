"""The feed-forward half of a layer, the part that needs no GPU: struct layouts, refusals, workspaces of refused calls."""
from __future__ import annotations

import ctypes
import math
import pathlib
import subprocess

import pytest

from geometricelementaryoperators_b200 import abi

ROOT = pathlib.Path(__file__).resolve().parent.parent
INVALID = 1
ref = ctypes.byref


def some(i):
    """Distinct addresses, never dereferenced: every call here is refused before its arrays are looked at."""
    return ctypes.c_void_p((i + 1) << 24)


def test_struct_layouts(tmp_path):
    names = {"geo_b200_block_norm_config_t": abi.BlockNormConfig, "geo_b200_gradient_t": abi.Gradient,
             "geo_b200_feed_forward_config_t": abi.FeedForwardConfig}
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


def test_enumerations():
    text = (ROOT / "include/geo/geo_b200.h").read_text()
    for prefix, names in (("ACTIVATION", ("SILU", "GELU", "SIGMOID", "RELU")),
                          ("GATE", ("NONE", "LINEAR", "SIGMOID", "TANH"))):
        for n in names:
            assert f"GEO_B200_{prefix}_{n} = {getattr(abi, f'{prefix}_{n}')}" in text


def feed_config(**k):
    d = dict(type=abi.BF16, gradient_type=abi.BF16, activation=abi.ACTIVATION_SILU, rows=16, cols=64, hidden=128)
    d.update(k)
    return abi.FeedForwardConfig(**d)


BAD_FEED = [dict(type=0), dict(type=5), dict(gradient_type=abi.F16), dict(gradient_type=abi.F64),
            dict(type=abi.F64, gradient_type=abi.F32), dict(activation=0), dict(activation=5), dict(reserved=1),
            dict(rows=0), dict(cols=0), dict(hidden=0), dict(rows=(1 << 24) + 1), dict(cols=(1 << 20) + 1),
            dict(hidden=(1 << 20) + 1), dict(x_stride=63), dict(gate_weight_stride=63), dict(up_weight_stride=63),
            dict(down_weight_stride=127), dict(gate_stride=127), dict(up_stride=127), dict(x_stride=1 << 60)]
FORWARD = [some(i) for i in range(8)]
VJP = [some(i) for i in range(12)]


@pytest.mark.parametrize("bad", BAD_FEED)
def test_feed_forward_refusals(bad):
    L, c = abi.lib(), feed_config(**bad)
    assert L.geo_b200_feed_forward_workspace(ref(c)) == 0
    assert L.geo_b200_feed_forward_vjp_workspace(ref(c)) == 0
    assert L.geo_b200_feed_forward(ref(c), *FORWARD, 1 << 40, None) == INVALID
    assert L.geo_b200_feed_forward_vjp(ref(c), *VJP, 1 << 40, None) == INVALID


def test_feed_forward_strides_of_the_other_direction():
    """A stride that only the other direction uses does not matter."""
    L = abi.lib()
    assert L.geo_b200_feed_forward_workspace(ref(feed_config(y_stride=63))) == 0
    assert L.geo_b200_feed_forward_vjp_workspace(ref(feed_config(y_stride=63))) > 0
    for name in ("y_cotangent_stride", "x_cotangent_stride"):
        assert L.geo_b200_feed_forward_workspace(ref(feed_config(**{name: 63}))) > 0
        assert L.geo_b200_feed_forward_vjp_workspace(ref(feed_config(**{name: 63}))) == 0


def test_feed_forward_null_arguments():
    L, c = abi.lib(), feed_config()
    assert L.geo_b200_feed_forward_workspace(None) == 0 and L.geo_b200_feed_forward_vjp_workspace(None) == 0
    assert L.geo_b200_feed_forward(None, *FORWARD, 1 << 40, None) == INVALID
    for missing in (0, 1, 2, 3, 4, 5, 6, 7):  # gate and up go together
        args = list(FORWARD)
        args[missing] = None
        assert L.geo_b200_feed_forward(ref(c), *args, 1 << 40, None) == INVALID
    for missing in (0, 1, 2, 3, 4, 5, 6, 11):
        args = list(VJP)
        args[missing] = None
        assert L.geo_b200_feed_forward_vjp(ref(c), *args, 1 << 40, None) == INVALID
    assert L.geo_b200_feed_forward_vjp(ref(c), *VJP[:7], None, None, None, None, VJP[11], 1 << 40, None) == INVALID
    need = L.geo_b200_feed_forward_workspace(ref(c))
    assert need >= 16 * 128 * 2
    assert L.geo_b200_feed_forward(ref(c), *FORWARD, need - 1, None) == INVALID
    need = L.geo_b200_feed_forward_vjp_workspace(ref(c))
    assert need >= 3 * 16 * 128 * 2
    assert L.geo_b200_feed_forward_vjp(ref(c), *VJP, need - 1, None) == INVALID
    for out, source in ((6, 0), (4, 3), (5, 4), (7, 0)):  # an output that is an input or another output
        args = list(FORWARD)
        args[out] = args[source]
        assert L.geo_b200_feed_forward(ref(c), *args, 1 << 40, None) == INVALID


def test_feed_forward_workspace_grows_with_copies():
    """16-bit rows off 16 bytes are copied; two-term inner values double their part."""
    L = abi.lib()
    plain = L.geo_b200_feed_forward_workspace(ref(feed_config()))
    odd = L.geo_b200_feed_forward_workspace(ref(feed_config(x_stride=65, gate_weight_stride=65)))
    assert odd >= plain + 2 * 64 * 16 + 2 * 64 * 128
    few = L.geo_b200_feed_forward_workspace(ref(feed_config(rows=2, gate_weight_stride=65)))
    assert few <= plain
    plain = L.geo_b200_feed_forward_vjp_workspace(ref(feed_config()))
    assert L.geo_b200_feed_forward_vjp_workspace(ref(feed_config(gradient_type=abi.F32))) >= plain + 3 * 2 * 16 * 128


def norm_config(**k):
    d = dict(type=abi.F32, parameter_type=abi.F32, rows=8, cols=64, epsilon=1e-5)
    d.update(k)
    return abi.LayerNormConfig(**d)


BAD_NORM = [dict(type=0), dict(type=5), dict(parameter_type=0), dict(parameter_type=abi.F64),
            dict(type=abi.F64, parameter_type=abi.F32), dict(type=abi.BF16, parameter_type=abi.F16),
            dict(rows=0), dict(cols=0), dict(cols=(1 << 24) + 1), dict(rows=(1 << 32) + 1),
            dict(epsilon=-1e-5), dict(epsilon=math.nan), dict(epsilon=math.inf), dict(x_stride=63),
            dict(x_stride=1 << 60)]


@pytest.mark.parametrize("bad", BAD_NORM)
def test_rms_norm_refusals(bad):
    L, c = abi.lib(), norm_config(**bad)
    assert L.geo_b200_rms_norm(ref(c), some(0), some(1), some(2), some(3), None) == INVALID
    assert L.geo_b200_rms_norm_vjp_workspace(ref(c)) == 0
    assert L.geo_b200_rms_norm_vjp(ref(c), *[some(i) for i in range(7)], 1 << 30, None) == INVALID


def test_rms_norm_null_arguments():
    L, c = abi.lib(), norm_config()
    assert L.geo_b200_rms_norm(None, some(0), None, some(1), None, None) == INVALID
    assert L.geo_b200_rms_norm(ref(c), None, None, some(1), None, None) == INVALID
    assert L.geo_b200_rms_norm(ref(c), some(0), None, None, None, None) == INVALID
    args = [some(i) for i in range(7)]
    for missing in (0, 2, 3):
        bad = list(args)
        bad[missing] = None
        assert L.geo_b200_rms_norm_vjp(ref(c), *bad, 1 << 30, None) == INVALID
    bad = list(args)
    bad[4] = bad[5] = None
    assert L.geo_b200_rms_norm_vjp(ref(c), *bad, 1 << 30, None) == INVALID
    assert L.geo_b200_rms_norm_vjp_workspace(None) == 0
    assert L.geo_b200_rms_norm_vjp_workspace(ref(c)) >= 64 * 4
    moved = norm_config(x_stride=64, y_stride=72)
    assert L.geo_b200_rms_norm(ref(moved), some(0), None, some(0), None, None) == INVALID


def block_config(**k):
    d = dict(type=abi.F32, parameter_type=abi.F32, gate=abi.GATE_SIGMOID, rows=8, cols=64, epsilon=1e-5,
             residual_scale=1.0, block_scale=0.5)
    d.update(k)
    return abi.BlockNormConfig(**d)


BLOCK = [some(i) for i in range(9)]
BLOCK_VJP = [some(i) for i in range(15)]


@pytest.mark.parametrize("bad", BAD_NORM + [dict(gate=4), dict(reserved=1), dict(residual_scale=math.inf),
                                            dict(block_scale=math.nan), dict(gate_stride=63), dict(z_stride=63)])
def test_block_norm_refusals(bad):
    L, c = abi.lib(), block_config(**bad)
    assert L.geo_b200_block_norm(ref(c), *BLOCK, None) == INVALID
    assert L.geo_b200_block_norm_vjp_workspace(ref(c)) == 0
    assert L.geo_b200_block_norm_vjp(ref(c), *BLOCK_VJP, 1 << 30, None) == INVALID


def test_block_norm_null_arguments():
    L, c = abi.lib(), block_config()
    for missing in (0, 1, 2, 5, 6):
        args = list(BLOCK)
        args[missing] = None
        assert L.geo_b200_block_norm(ref(c), *args, None) == INVALID
    plain = block_config(gate=abi.GATE_NONE)
    assert L.geo_b200_block_norm(ref(plain), *BLOCK, None) == INVALID  # a gate that is not used
    args = list(BLOCK)
    args[6] = args[5]  # y and z in one array
    assert L.geo_b200_block_norm(ref(c), *args, None) == INVALID
    for missing in (0, 1, 2, 5, 6, 7):
        args = list(BLOCK_VJP)
        args[missing] = None
        assert L.geo_b200_block_norm_vjp(ref(c), *args, 1 << 30, None) == INVALID
    args = list(BLOCK_VJP)
    args[1] = None
    assert L.geo_b200_block_norm_vjp(ref(plain), *args, 1 << 30, None) == INVALID  # gate_bar without a gate
    args = list(BLOCK_VJP)
    args[9] = args[10] = args[11] = args[12] = args[13] = None
    assert L.geo_b200_block_norm_vjp(ref(c), *args, 1 << 30, None) == INVALID
    args = list(BLOCK_VJP)
    args[10] = args[9]  # two outputs in one array
    assert L.geo_b200_block_norm_vjp(ref(c), *args, 1 << 30, None) == INVALID
    assert L.geo_b200_block_norm_vjp_workspace(None) == 0
    assert L.geo_b200_block_norm_vjp_workspace(ref(c)) >= 2 * 64 * 4


def table(*entries):
    return (abi.Gradient * len(entries))(*[abi.Gradient(**{"type": abi.F32, "count": 64, **e}) for e in entries])


@pytest.mark.parametrize("bad", [dict(type=0), dict(type=5), dict(reserved=1), dict(count=(1 << 40) + 1)])
def test_gradient_clip_refusals(bad):
    L, t = abi.lib(), table(dict(gradient=1 << 24, clipped=1 << 24, **bad))
    assert L.geo_b200_gradient_clip_workspace(t, 1) == 0
    assert L.geo_b200_gradient_clip(t, 1, 1.0, None, None, some(9), 1 << 20, None) == INVALID


def test_gradient_clip_arguments():
    L, t = abi.lib(), table(dict(gradient=1 << 24, clipped=1 << 24))
    call = L.geo_b200_gradient_clip
    assert L.geo_b200_gradient_clip_workspace(None, 1) == 0 and L.geo_b200_gradient_clip_workspace(t, 0) == 0
    assert L.geo_b200_gradient_clip_workspace(t, 65537) == 0
    need = L.geo_b200_gradient_clip_workspace(t, 1)
    assert need >= 24
    for bad in (0.0, -1.0, math.nan):
        assert call(t, 1, bad, None, None, some(9), 1 << 20, None) == INVALID
    assert call(None, 1, 1.0, None, None, some(9), 1 << 20, None) == INVALID
    assert call(t, 0, 1.0, None, None, some(9), 1 << 20, None) == INVALID
    assert call(t, 1, 1.0, None, None, None, 1 << 20, None) == INVALID
    assert call(t, 1, 1.0, None, None, some(9), need - 1, None) == INVALID
    assert call(table(dict(gradient=None)), 1, 1.0, None, None, some(9), 1 << 20, None) == INVALID
