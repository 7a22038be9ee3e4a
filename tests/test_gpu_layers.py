"""Layer operators on the GPU against their 64-bit definitions (layer_reference.py), with bounds counted in
roundings: sizes from one row and one value on, every type, strided and misaligned arrays, arrays in place,
non-finite values, captured graphs, and gradients against differences."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import layer_reference as ref
from geometricelementaryoperators_b200 import abi
from gpu_helpers import stream, torch

pytestmark = pytest.mark.gpu

INVALID = 1
EPS = 1e-5


def call(name, *args):
    assert getattr(abi.lib(), name)(*args, stream()) == 0, name


def make(rows, cols, dtype, pad=0, seed=0, shift=0.0, size=1.0):
    """[rows][cols] on the GPU; `pad` > 0: a slice that starts `pad` values into rows of cols + 2 pad."""
    t = torch()
    g = t.Generator(device="cuda").manual_seed(seed)
    v = t.randn(rows, cols + 2 * pad, generator=g, device="cuda", dtype=t.float64) * size + shift
    return v.to(dtype)[:, pad:pad + cols]


def like(x, fill=7.0):
    """An output of x's shape and strides in a buffer filled with `fill`, and that buffer."""
    t = torch()
    stride = x.stride(0) if x.shape[0] > 1 else x.shape[1]
    pad = (stride - x.shape[1]) // 2
    whole = t.full((x.shape[0], stride), fill, device="cuda", dtype=x.dtype)
    return whole[:, pad:pad + x.shape[1]], whole


def untouched(whole, cols, fill=7.0):
    pad = (whole.shape[1] - cols) // 2
    return bool((whole[:, :pad] == fill).all()) and bool((whole[:, pad + cols:] == fill).all())


def norm_config(x, ptype, **k):
    s = x.stride(0) if x.shape[0] > 1 else 0
    d = dict(type=TYPE[x.dtype], parameter_type=TYPE[ptype], rows=x.shape[0], cols=x.shape[1], x_stride=s, y_stride=s,
             y_cotangent_stride=s, x_cotangent_stride=s, epsilon=EPS)
    d.update(k)
    return abi.LayerNormConfig(**d)


def drop_config(x, rate=0.3, dimension=0, seed=0x123456789ABCDEF0, offset=(1 << 40) + 5, **k):
    s = x.stride(0) if x.shape[0] > 1 else 0
    d = dict(type=TYPE[x.dtype], dimension=dimension, rows=x.shape[0], cols=x.shape[1], x_stride=s, residual_stride=s,
             y_stride=s, y_cotangent_stride=s, x_cotangent_stride=s, rate=rate, seed=seed, offset=offset)
    d.update(k)
    return abi.DropoutConfig(**d)


class _Types(dict):
    def __missing__(self, dtype):
        return {ref.torch_type(n): c for n, c in ref.TYPES.items()}[dtype]


TYPE = _Types()
P = ref.pointer


def mask(c, first_row=0, rows=None):
    t = torch()
    m = ref.kept(c.rows if rows is None else rows, c.cols, c.dimension, c.rate, c.seed, c.offset, first_row)
    return t.from_numpy(m).cuda()


def parameters(cols, ptype, seed=9):
    t = torch()
    g = t.Generator(device="cuda").manual_seed(seed)
    return ((1 + 0.3 * t.randn(cols, generator=g, device="cuda")).to(ptype),
            (0.5 * t.randn(cols, generator=g, device="cuda")).to(ptype))


def stats_like(x):
    t = torch()
    return [t.full((x.shape[0],), 7.0, device="cuda", dtype=ref.wide_type(x.dtype)) for _ in range(2)]


def workspace(c):
    size = abi.lib().geo_b200_layer_norm_vjp_workspace(ctypes.byref(c))
    assert size > 0
    return torch().empty(size, device="cuda", dtype=torch().uint8), size


# (type, type of the parameters)
KINDS = [("f64", "f64"), ("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]
# (rows, cols, pad): single values, odd lengths, slices off 16-byte boundaries, one row, many rows, long rows.
SHAPES = [(1, 1, 0), (3, 1, 0), (5, 7, 0), (1, 64, 0), (130, 64, 0), (1, 1024, 0), (33, 96, 1), (9, 333, 0), (7, 1000, 8),
          (300, 128, 0), (17, 2056, 0), (40, 1003, 1), (3, 5120, 0), (2, 8192, 0), (5, 16384, 0), (2, 16381, 3),
          (2000, 40, 0), (4100, 16, 0), (6, 20008, 0), (700, 257, 0)]
# Many rows for every team of threads, so that each takes several: part of a block, a block, clusters of 2 to 8 blocks.
LONG = [(4100, 520, 0), (3001, 1003, 1), (1500, 4096, 0), (1300, 4001, 1), (1000, 5120, 0), (701, 16384, 0), (900, 8193, 1),
        (333, 32768, 0)]


@pytest.mark.parametrize("kind,pkind", KINDS)
@pytest.mark.parametrize("rows,cols,pad", SHAPES + LONG)
def test_layer_norm(kind, pkind, rows, cols, pad):
    dtype, ptype = ref.torch_type(kind), ref.torch_type(pkind)
    x = make(rows, cols, dtype, pad, seed=cols, shift=0.5)
    w, b = parameters(cols, ptype)
    y, whole = like(x)
    mean, rstd = stats_like(x)
    c = norm_config(x, ptype)
    call("geo_b200_layer_norm", ctypes.byref(c), P(x), P(w), P(b), P(y), P(mean), P(rstd))
    want = ref.norm(x.double(), w.double(), b.double(), EPS)
    bounds = ref.norm_bound(x.double(), w.double(), b.double(), want[2], want[0], dtype, max(ref.PATH, cols // 100))
    for got, v, bound, what in zip((y, mean, rstd), want, bounds, ("y", "mean", "rstd")):
        ref.assert_within(got, v, bound, what)
    assert untouched(whole, cols)
    again, _ = like(x)
    call("geo_b200_layer_norm", ctypes.byref(c), P(x), P(w), P(b), P(again), None, None)
    assert torch().equal(again, y)


@pytest.mark.parametrize("kind,pkind", KINDS)
@pytest.mark.parametrize("rows,cols,pad", SHAPES + LONG)
def test_layer_norm_vjp(kind, pkind, rows, cols, pad):
    t = torch()
    dtype, ptype = ref.torch_type(kind), ref.torch_type(pkind)
    x, dy = make(rows, cols, dtype, pad, seed=cols, shift=0.5), make(rows, cols, dtype, pad, seed=cols + 1)
    w, b = parameters(cols, ptype)
    _, mean, rstd = ref.norm(x.double(), None, None, EPS)
    mean, rstd = mean.to(ref.wide_type(dtype)), rstd.to(ref.wide_type(dtype))
    dx, whole = like(x)
    dw, db = t.full_like(w, 7.0), t.full_like(b, 7.0)
    c = norm_config(x, ptype)
    space, size = workspace(c)
    call("geo_b200_layer_norm_vjp", ctypes.byref(c), P(x), P(w), P(mean), P(rstd), P(dy), P(dx), P(dw), P(db), P(space),
         size)
    wide = [v.double() for v in (x, w, mean, rstd, dy)]
    want = ref.norm_vjp(*wide)
    bounds = ref.norm_vjp_bound(*wide, want[0], dtype, max(ref.PATH, cols // 100))
    ref.assert_within(dx, want[0], bounds[0], "dx")
    u = ref.half_step(ptype)
    ref.assert_within(dw, want[1], bounds[1] + u * want[1].abs() + ref.least(ptype), "dweight")
    ref.assert_within(db, want[2], bounds[2] + u * want[2].abs() + ref.least(ptype), "dbias")
    assert untouched(whole, cols)
    # Each output alone, and without a weight; the same values as together.
    only, _ = like(x)
    call("geo_b200_layer_norm_vjp", ctypes.byref(c), P(x), P(w), P(mean), P(rstd), P(dy), P(only), None, None, None, 0)
    assert t.equal(only, dx)
    dw2, db2 = t.empty_like(w), t.empty_like(b)
    call("geo_b200_layer_norm_vjp", ctypes.byref(c), P(x), P(w), P(mean), P(rstd), P(dy), None, P(dw2), None, P(space),
         size)
    call("geo_b200_layer_norm_vjp", ctypes.byref(c), P(x), P(w), P(mean), P(rstd), P(dy), None, None, P(db2), P(space),
         size)
    for got, v, bound in ((dw2, want[1], bounds[1]), (db2, want[2], bounds[2])):
        ref.assert_within(got, v, bound + u * v.abs() + ref.least(ptype))
    plain = ref.norm_vjp(wide[0], None, *wide[2:])
    call("geo_b200_layer_norm_vjp", ctypes.byref(c), P(x), None, P(mean), P(rstd), P(dy), P(only), P(dw2), P(db2),
         P(space), size)
    ref.assert_within(only, plain[0], ref.norm_vjp_bound(wide[0], None, *wide[2:], plain[0], dtype,
                                                         max(ref.PATH, cols // 100))[0], "dx without weight")


@pytest.mark.parametrize("kind", ["f64", "f32", "bf16"])
@pytest.mark.parametrize("cols,pad", [(64, 0), (1000, 0), (333, 1), (20000, 0)])
def test_layer_norm_in_place_and_without_parameters(kind, cols, pad):
    dtype = ref.torch_type(kind)
    x = make(37, cols, dtype, pad, shift=-2.0)
    want, _ = like(x)
    c = norm_config(x, dtype)
    call("geo_b200_layer_norm", ctypes.byref(c), P(x), None, None, P(want), None, None)
    exact = ref.norm(x.double(), None, None, EPS)
    ref.assert_within(want, exact[0], ref.norm_bound(x.double(), None, None, exact[2], exact[0], dtype,
                                                     max(ref.PATH, cols // 100))[0])
    w, b = parameters(cols, dtype)
    only_bias, _ = like(x)
    call("geo_b200_layer_norm", ctypes.byref(c), P(x), None, P(b), P(only_bias), None, None)
    ref.assert_within(only_bias, exact[0] + b.double(), ref.norm_bound(
        x.double(), None, b.double(), exact[2], exact[0] + b.double(), dtype, max(ref.PATH, cols // 100))[0])
    same = x.clone() if pad == 0 else x
    call("geo_b200_layer_norm", ctypes.byref(c), P(same), None, None, P(same), None, None)
    assert torch().equal(same, want)
    # The VJP over its cotangent and over x.
    x, dy = make(37, cols, dtype, pad, shift=-2.0), make(37, cols, dtype, pad, seed=5)
    mean, rstd = exact[1].to(ref.wide_type(dtype)), exact[2].to(ref.wide_type(dtype))
    space, size = workspace(c)
    outs = []
    for target in ("apart", "dy", "x"):
        a, d = like(x)[0].copy_(x), like(x)[0].copy_(dy)
        o = {"apart": like(x)[0], "dy": d, "x": a}[target]
        dw, db = torch().empty_like(w), torch().empty_like(b)
        call("geo_b200_layer_norm_vjp", ctypes.byref(c), P(a), P(w), P(mean), P(rstd), P(d), P(o), P(dw), P(db),
             P(space), size)
        outs.append((o.clone(), dw, db))
    for o in outs[1:]:
        assert all(torch().equal(p, q) for p, q in zip(outs[0], o))


@pytest.mark.parametrize("kind,pkind", KINDS)
@pytest.mark.parametrize("cols", [8, 72, 1000, 5120])
def test_layer_norm_parameters_off_16_bytes(kind, pkind, cols):
    """Weight, bias and their cotangents start one value into their arrays: the values of aligned ones, in the bounds."""
    t = torch()
    dtype, ptype = ref.torch_type(kind), ref.torch_type(pkind)
    x, dy = make(37, cols, dtype, seed=1), make(37, cols, dtype, seed=2)
    w, b = (v[1:] for v in parameters(cols + 1, ptype))
    y, _ = like(x)
    mean, rstd = stats_like(x)
    c = norm_config(x, ptype)
    call("geo_b200_layer_norm", ctypes.byref(c), P(x), P(w), P(b), P(y), P(mean), P(rstd))
    want = ref.norm(x.double(), w.double(), b.double(), EPS)
    ref.assert_within(y, want[0], ref.norm_bound(x.double(), w.double(), b.double(), want[2], want[0], dtype)[0])
    space, size = workspace(c)
    whole = t.full((2, cols + 2), 7.0, device="cuda", dtype=ptype)
    dw, db = whole[0, 1:-1], whole[1, 1:-1]
    dx, _ = like(x)
    call("geo_b200_layer_norm_vjp", ctypes.byref(c), P(x), P(w), P(mean), P(rstd), P(dy), P(dx), P(dw), P(db), P(space),
         size)
    wide = [v.double() for v in (x, w, mean, rstd, dy)]
    want = ref.norm_vjp(*wide)
    bounds = ref.norm_vjp_bound(*wide, want[0], dtype)
    u = ref.half_step(ptype)
    ref.assert_within(dx, want[0], bounds[0], "dx")
    ref.assert_within(dw, want[1], bounds[1] + u * want[1].abs() + ref.least(ptype), "dweight")
    ref.assert_within(db, want[2], bounds[2] + u * want[2].abs() + ref.least(ptype), "dbias")
    assert (whole[:, 0] == 7).all() and (whole[:, -1] == 7).all()


@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,pads", [(50, 100, (1, 0, 3, 2)), (9, 1003, (0, 5, 1, 2)), (40, 64, (8, 1, 0, 4)),
                                            (7, 5001, (2, 3, 0, 1)), (130, 13, (0, 1, 2, 3))])
def test_arrays_of_unlike_alignment(kind, rows, cols, pads):
    """Each array with a stride and an alignment of its own: the bits of packed arrays' dropout, the fused call and its
    VJP within their bounds, and nothing written beside the rows."""
    t = torch()
    dtype = ref.torch_type(kind)
    x, res, dy, dz = (make(rows, cols, dtype, p, seed=i) for i, p in enumerate(pads))
    packed = [v.contiguous() for v in (x, res, dy, dz)]
    w, b = parameters(cols, dtype)
    strides = [v.stride(0) for v in (x, res, dy, dz)]
    outs = [like(v) for v in (res, dy, dz, x)]  # z, y, dresidual, dx
    so = [strides[1], strides[2], strides[3], strides[0]]
    d = drop_config(x, 0.3, x_stride=strides[0], residual_stride=strides[1], y_stride=so[0],
                    y_cotangent_stride=strides[3], x_cotangent_stride=so[3])
    n = norm_config(x, dtype, x_stride=so[0], y_stride=so[1], y_cotangent_stride=strides[2], x_cotangent_stride=so[2])
    dp, np_ = drop_config(packed[0], 0.3), norm_config(packed[0], dtype)
    z, _ = like(packed[0])
    call("geo_b200_dropout", ctypes.byref(d), P(x), P(res), None, P(outs[0][0]))
    call("geo_b200_dropout", ctypes.byref(dp), P(packed[0]), P(packed[1]), None, P(z))
    assert t.equal(outs[0][0], z)
    mean, rstd = stats_like(x)
    call("geo_b200_residual_dropout_layer_norm", ctypes.byref(n), ctypes.byref(d), P(x), P(res), None, P(w), P(b),
         P(outs[0][0]), P(outs[1][0]), P(mean), P(rstd))
    assert t.equal(outs[0][0], z)
    keep = mask(dp)
    exact_z = drop_reference(packed[0].double(), packed[1].double(), keep, 0.3)
    want = ref.norm(exact_z, w.double(), b.double(), EPS)
    bound = ref.norm_bound(exact_z, w.double(), b.double(), want[2], want[0], dtype, 2 * ref.PATH)[0]
    ref.assert_within(outs[1][0], want[0], bound, "y")
    space, size = workspace(n)
    dw, db = t.empty_like(w), t.empty_like(b)
    call("geo_b200_residual_dropout_layer_norm_vjp", ctypes.byref(n), ctypes.byref(d), None, P(outs[0][0]), P(w), P(mean),
         P(rstd), P(dy), P(dz), P(outs[2][0]), P(outs[3][0]), P(dw), P(db), P(space), size)
    wide = [v.double() for v in (z, w, mean, rstd, packed[2])]
    norm_dx, want_dw, want_db = ref.norm_vjp(*wide)
    total = norm_dx + packed[3].double()
    bounds = ref.norm_vjp_bound(*wide, total, dtype)
    ref.assert_within(outs[2][0], total, bounds[0] + ref.u_wide(dtype) * total.abs(), "dresidual")
    assert bool((outs[3][0][~keep] == 0).all())
    u = ref.half_step(dtype)
    ref.assert_within(dw, want_dw, bounds[1] + u * want_dw.abs() + ref.least(dtype), "dweight")
    ref.assert_within(db, want_db, bounds[2] + u * want_db.abs() + ref.least(dtype), "dbias")
    for _, whole in outs:
        assert untouched(whole, cols)


@pytest.mark.parametrize("cols", [16, 100, 1024, 5000, 20000])
def test_layer_norm_far_from_zero(cols):
    """Rows whose mean is 1000 times their spread: the statistics are those about the row's own mean."""
    dtype = torch().float32
    x = make(21, cols, dtype, shift=1000.0)
    y, _ = like(x)
    mean, rstd = stats_like(x)
    call("geo_b200_layer_norm", ctypes.byref(norm_config(x, dtype)), P(x), None, None, P(y), P(mean), P(rstd))
    want = ref.norm(x.double(), None, None, EPS)
    bounds = ref.norm_bound(x.double(), None, None, want[2], want[0], dtype, max(ref.PATH, cols // 100))
    for got, v, b in zip((y, mean, rstd), want, bounds):
        ref.assert_within(got, v, b)


@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("cols", [5, 64, 1000, 20000])
def test_layer_norm_non_finite_rows_stay_apart(kind, cols):
    t = torch()
    dtype = ref.torch_type(kind)
    x = make(9, cols, dtype)
    x[2, 3] = float("nan")
    x[5, 1] = float("inf")
    x[6] = 3.0  # variance 0
    c = norm_config(x, dtype)
    y, _ = like(x)
    call("geo_b200_layer_norm", ctypes.byref(c), P(x), None, None, P(y), None, None)
    bad = t.isnan(y).any(1).cpu().tolist()
    assert bad == [i in (2, 5) for i in range(9)]
    assert t.isnan(y[2]).all() and t.isnan(y[5]).all() and (y[6] == 0).all()


def test_layer_norm_rows_past_32_bits():
    """Rows further than 2^32 values from the first one, in an array of 8.6 GB of which three rows are used."""
    t = torch()
    stride, cols = (1 << 31) + 64, 1000
    whole = t.empty(2 * stride + cols, device="cuda", dtype=t.bfloat16)
    x = t.as_strided(whole, (3, cols), (stride, 1))
    x.copy_(make(3, cols, t.bfloat16))
    packed = x.contiguous()
    w, b = parameters(cols, t.float32)
    y, _ = like(packed)
    c = norm_config(packed, t.float32, x_stride=stride, y_stride=0, y_cotangent_stride=0, x_cotangent_stride=stride)
    call("geo_b200_layer_norm", ctypes.byref(c), P(whole), P(w), P(b), P(y), None, None)
    want, _ = like(packed)
    call("geo_b200_layer_norm", ctypes.byref(norm_config(packed, t.float32)), P(packed), P(w), P(b), P(want), None, None)
    assert t.equal(y, want)
    drop = drop_config(packed, y_stride=stride, x_stride=stride)
    call("geo_b200_dropout", ctypes.byref(drop), P(whole), None, None, P(whole))
    call("geo_b200_dropout", ctypes.byref(drop_config(packed)), P(packed), None, None, P(want))
    assert t.equal(x, want)


# ---- dropout ------------------------------------------------------------------


def drop_reference(x, residual, keep, rate):
    t = torch()
    z = t.where(keep, x * ref.scale(rate), t.zeros_like(x))
    return z + residual if residual is not None else z


def drop_bound(x, keep, rate, z, dtype):
    """The scale's rounding, the product's and the sum's (of a sum no larger than the result and the product)."""
    u = ref.u_wide(dtype)
    return ref.half_step(dtype) * z.abs() + ref.least(dtype) + u * (4 * ref.scale(rate) * x.abs() * keep + z.abs())


@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,pad,dimension", [
    (1, 1, 0, 0), (1, 7, 0, 0), (3, 1, 0, 0), (5, 64, 0, 6), (5, 64, 0, 0), (33, 96, 1, 0), (33, 96, 1, 3), (9, 333, 0, 0),
    (7, 1000, 8, 2), (130, 1003, 1, 0), (300, 128, 0, 5), (4, 2056, 3, 1), (50, 4096, 0, 0), (64, 192, 4, 6),
    (1000, 24, 0, 3), (1, 100000, 0, 4)])
def test_dropout(kind, rows, cols, pad, dimension):
    t = torch()
    dtype = ref.torch_type(kind)
    x, res = make(rows, cols, dtype, pad, seed=3), make(rows, cols, dtype, pad, seed=4)
    for rate in (0.3, 0.0):
        c = drop_config(x, rate, dimension)
        keep = mask(c)
        for residual in (None, res):
            y, whole = like(x)
            call("geo_b200_dropout", ctypes.byref(c), P(x), P(residual), None, P(y))
            want = drop_reference(x.double(), None if residual is None else residual.double(), keep, rate)
            ref.assert_within(y, want, drop_bound(x.double(), keep, rate, want, dtype), f"rate {rate}")
            assert untouched(whole, cols)
        dx, whole = like(x)
        call("geo_b200_dropout_vjp", ctypes.byref(c), None, P(x), P(dx))
        want = drop_reference(x.double(), None, keep, rate)
        ref.assert_within(dx, want, drop_bound(x.double(), keep, rate, want, dtype), "vjp")
        assert untouched(whole, cols)
    for over in ("x", "residual"):  # in place
        a, r = like(x)[0].copy_(x), like(x)[0].copy_(res)
        y, _ = like(x)
        c = drop_config(x, 0.5, dimension)
        call("geo_b200_dropout", ctypes.byref(c), P(a), P(r), None, P(y))
        o = a if over == "x" else r
        call("geo_b200_dropout", ctypes.byref(c), P(a), P(r), None, P(o))
        assert t.equal(o, y)


def test_dropout_strides_do_not_enter_the_mask():
    t = torch()
    x = make(40, 1000, t.float32, 1).fill_(1.0)
    c = drop_config(x)
    y, _ = like(x)
    call("geo_b200_dropout", ctypes.byref(c), P(x), None, None, P(y))
    packed = x.contiguous()
    z, _ = like(packed)
    call("geo_b200_dropout", ctypes.byref(drop_config(packed)), P(packed), None, None, P(z))
    assert t.equal(y, z)


def test_dropout_rate_ends_and_dropped_values():
    t = torch()
    x = make(30, 256, t.float32)
    c = drop_config(x, 0.5)
    keep = mask(c)
    x[~keep] = float("nan")  # what is dropped does not matter
    res = make(30, 256, t.float32, seed=8)
    y, _ = like(x)
    call("geo_b200_dropout", ctypes.byref(c), P(x), P(res), None, P(y))
    assert t.equal(y[~keep], res[~keep]) and not t.isnan(y).any()
    for rate in (1.0, 1.0 - 2.0 ** -18):
        call("geo_b200_dropout", ctypes.byref(drop_config(x, rate)), P(x), None, None, P(y))
        assert (y == 0).all()
    x = make(30, 256, t.float32)
    call("geo_b200_dropout", ctypes.byref(drop_config(x, 2.0 ** -18)), P(x), None, None, P(y))
    assert t.equal(x, y)


def test_dropout_counts_and_seeds():
    """Kept shares of 2^22 draws within five standard deviations; other seeds and offsets draw other masks."""
    t = torch()
    x = t.ones(1 << 11, 1 << 11, device="cuda")
    seen = []
    for seed, offset in ((1, 0), (2, 0), (1, 1), (1, 1 << 32), (1 << 32, 0)):
        y, _ = like(x)
        call("geo_b200_dropout", ctypes.byref(drop_config(x, 0.25, seed=seed, offset=offset)), P(x), None, None, P(y))
        share = float((y != 0).double().mean())
        assert abs(share - 0.75) <= 5 * (0.25 * 0.75 / 2 ** 22) ** 0.5
        seen.append(y != 0)
    for i in range(len(seen)):
        for j in range(i):
            both = float((seen[i] & seen[j]).double().mean())
            assert abs(both - 0.5625) <= 5 * (0.5625 * 0.4375 / 2 ** 22) ** 0.5


def test_dropout_units_past_32_bits():
    """More than 2^32 units: the last rows of 4.3e9 values, one unit each."""
    t = torch()
    cols = 1 << 16
    rows = (1 << 16) + 3
    x = t.ones(rows, cols, device="cuda", dtype=t.bfloat16)
    c = drop_config(x, 0.5)
    call("geo_b200_dropout", ctypes.byref(c), P(x), None, None, P(x))
    for first in (0, rows - 4):
        assert t.equal(x[first:first + 4] != 0, mask(c, first, 4))


# ---- residual + dropout + layer norm --------------------------------------------

FUSED = [(1, 1, 0, 0), (3, 7, 0, 0), (1, 1024, 0, 0), (130, 64, 0, 6), (33, 96, 1, 3), (9, 333, 0, 0), (7, 1000, 8, 2),
         (300, 128, 0, 5), (40, 1003, 1, 0), (3, 5120, 0, 0), (5, 16384, 0, 1), (2, 16381, 3, 0), (6, 20008, 0, 3),
         (2000, 40, 0, 1), (700, 258, 0, 1), (4100, 520, 0, 3), (3001, 1003, 1, 0), (1500, 4096, 0, 0), (1000, 5120, 0, 6),
         (701, 16384, 0, 0), (900, 8193, 1, 0)]


@pytest.mark.parametrize("kind,pkind", KINDS)
@pytest.mark.parametrize("rows,cols,pad,dimension", FUSED)
def test_residual_dropout_layer_norm(kind, pkind, rows, cols, pad, dimension):
    t = torch()
    dtype, ptype = ref.torch_type(kind), ref.torch_type(pkind)
    x, res = make(rows, cols, dtype, pad, seed=1, size=0.5), make(rows, cols, dtype, pad, seed=2, shift=0.5)
    w, b = parameters(cols, ptype)
    for rate in (0.3, 0.0):
        n, d = norm_config(x, ptype), drop_config(x, rate, dimension)
        (z, zw), (y, yw) = like(x), like(x)
        mean, rstd = stats_like(x)
        call("geo_b200_residual_dropout_layer_norm", ctypes.byref(n), ctypes.byref(d), P(x), P(res), None, P(w), P(b),
             P(z), P(y), P(mean), P(rstd))
        keep = mask(d)
        want_z = drop_reference(x.double(), res.double(), keep, rate)
        ref.assert_within(z, want_z, drop_bound(x.double(), keep, rate, want_z, dtype), "z")
        want = ref.norm(want_z, w.double(), b.double(), EPS)
        # Each value of z carries 4 more roundings of its summands, each at most the average times cols / 4.
        path = max(ref.PATH, cols // 100)
        bounds = ref.norm_bound(want_z, w.double(), b.double(), want[2], want[0], dtype, path + 8)
        u = ref.u_wide(dtype)
        each = u * (4 * ref.scale(rate) * x.double().abs() * keep + want_z.abs())
        extra = (each + each.mean(1, keepdim=True)) * want[2][:, None]
        hat = (want_z - want[1][:, None]).abs() * want[2][:, None]
        extra = (extra + hat * (extra * hat).mean(1, keepdim=True)) * w.double().abs()
        ref.assert_within(y, want[0], bounds[0] + extra, "y")
        ref.assert_within(mean, want[1], bounds[1] + each.mean(1), "mean")
        ref.assert_within(rstd, want[2], bounds[2] + want[2] * ((each * hat).mean(1) * want[2]), "rstd")
        assert untouched(zw, cols) and untouched(yw, cols)
        # z over the residual, y over x.
        x2, r2 = like(x)[0].copy_(x), like(x)[0].copy_(res)
        call("geo_b200_residual_dropout_layer_norm", ctypes.byref(n), ctypes.byref(d), P(x2), P(r2), None, P(w), P(b),
             P(r2), P(x2), None, None)
        assert t.equal(r2, z) and t.equal(x2, y)


@pytest.mark.parametrize("kind,pkind", KINDS)
@pytest.mark.parametrize("rows,cols,pad,dimension", FUSED)
def test_residual_dropout_layer_norm_vjp(kind, pkind, rows, cols, pad, dimension):
    t = torch()
    dtype, ptype = ref.torch_type(kind), ref.torch_type(pkind)
    z, dy, dz = (make(rows, cols, dtype, pad, seed=s, shift=0.2) for s in (1, 2, 3))
    w, b = parameters(cols, ptype)
    _, mean, rstd = ref.norm(z.double(), None, None, EPS)
    mean, rstd = mean.to(ref.wide_type(dtype)), rstd.to(ref.wide_type(dtype))
    rate = 0.3
    n, d = norm_config(z, ptype), drop_config(z, rate, dimension)
    keep = mask(d)
    wide = [v.double() for v in (z, w, mean, rstd, dy)]
    norm_dx, want_dw, want_db = ref.norm_vjp(*wide)
    u = ref.half_step(ptype)
    space, size = workspace(n)
    saved = None
    for cotangent in (dz, None):
        (dres, rw), (dx, xw) = like(z), like(z)
        dw, db = t.full_like(w, 7.0), t.full_like(b, 7.0)
        call("geo_b200_residual_dropout_layer_norm_vjp", ctypes.byref(n), ctypes.byref(d), None, P(z), P(w), P(mean),
             P(rstd), P(dy), P(cotangent), P(dres), P(dx), P(dw), P(db), P(space), size)
        want = norm_dx if cotangent is None else norm_dx + dz.double()
        bounds = ref.norm_vjp_bound(*wide, want, dtype, max(ref.PATH, cols // 100))
        inner = bounds[0] - ref.half_step(dtype) * want.abs() + ref.u_wide(dtype) * want.abs()
        ref.assert_within(dres, want, bounds[0] + ref.u_wide(dtype) * want.abs(), "dresidual")
        want_dx = t.where(keep, want * ref.scale(rate), t.zeros_like(want))
        ref.assert_within(dx, want_dx, drop_bound(want, keep, rate, want_dx, dtype) + ref.scale(rate) * inner, "dx")
        ref.assert_within(dw, want_dw, bounds[1] + u * want_dw.abs() + ref.least(ptype), "dweight")
        ref.assert_within(db, want_db, bounds[2] + u * want_db.abs() + ref.least(ptype), "dbias")
        assert untouched(rw, cols) and untouched(xw, cols)
        saved = saved or (dres, dx, dw, db)
    # One output at a time, and outputs over the inputs.
    for which in (9, 10):
        outs = [None, None]
        outs[which - 9], _ = like(z)
        call("geo_b200_residual_dropout_layer_norm_vjp", ctypes.byref(n), ctypes.byref(d), None, P(z), P(w), P(mean),
             P(rstd), P(dy), P(dz), P(outs[0]), P(outs[1]), None, None, None, 0)
        assert t.equal(outs[which - 9], saved[which - 9])
    a, e, f = (like(z)[0].copy_(v) for v in (z, dy, dz))
    call("geo_b200_residual_dropout_layer_norm_vjp", ctypes.byref(n), ctypes.byref(d), None, P(a), P(w), P(mean),
         P(rstd), P(e), P(f), P(f), P(e), P(dw), P(db), P(space), size)
    assert all(t.equal(p, q) for p, q in zip((f, e, dw, db), saved))


# ---- rotary ---------------------------------------------------------------------


def rotary_case(kind, batch, tokens, heads, head_dim, order="bthd", pad=0, seed=0):
    """x as [batch][tokens][heads][head_dim], laid out in `order`, heads `pad` values apart."""
    t = torch()
    g = t.Generator(device="cuda").manual_seed(seed)
    sizes = {"b": batch, "t": tokens, "h": heads, "d": head_dim + pad}
    v = t.randn([sizes[c] for c in order], generator=g, device="cuda", dtype=t.float64).to(ref.torch_type(kind))
    return v.permute([order.index(c) for c in "bthd"])[..., :head_dim]


def rotary_shape(x, y, **k):
    d = dict(type=TYPE[x.dtype], position_type=abi.I64, batch=x.shape[0], tokens=x.shape[1], heads=x.shape[2],
             head_dim=x.shape[3], x_batch_stride=x.stride(0), x_token_stride=x.stride(1), x_head_stride=x.stride(2),
             y_batch_stride=y.stride(0), y_token_stride=y.stride(1), y_head_stride=y.stride(2))
    d.update(k)
    return abi.RotaryShape(**d)


def rotary_plan(rotary_dim, layout, amplitude=1.0, scaling="none", **k):
    kind = ["none", "linear", "base", "banded"].index(scaling)
    c = abi.RotaryConfig(layout=abi.ROTARY_HALF if layout == "half" else abi.ROTARY_INTERLEAVED, rotary_dim=rotary_dim,
                         base=10000.0, scaling=kind, factor=4.0, original_length=4096.0, low_rotations=1.0,
                         high_rotations=32.0, amplitude=amplitude)
    plan = abi.RotaryPlan()
    assert abi.lib().geo_b200_rotary_plan_init(ctypes.byref(plan), ctypes.byref(c)) == 0
    return plan, ref.rotary_turns(rotary_dim, 10000.0, scaling, 4.0, 4096.0, 1.0, 32.0)


@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("batch,tokens,heads,head_dim,rotary_dim,order,pad,scaling", [
    (1, 1, 1, 2, 2, "bthd", 0, "none"), (1, 1, 40, 128, 128, "bthd", 0, "none"), (8, 1, 5, 64, 64, "bthd", 0, "linear"),
    (2, 33, 3, 96, 64, "bthd", 0, "banded"), (2, 33, 3, 96, 64, "bhtd", 0, "banded"), (3, 7, 2, 80, 20, "bthd", 3, "base"),
    (1, 513, 1, 128, 128, "bthd", 0, "none"), (2, 5, 9, 256, 256, "bhtd", 8, "linear"), (2, 19, 4, 34, 6, "tbhd", 1, "none"),
    (1, 300, 12, 64, 32, "bthd", 0, "base"), (1, 70, 2, 300, 256, "hbtd", 0, "none"), (1, 3, 130, 16, 16, "bthd", 0, "none")])
def test_rotary(kind, layout, batch, tokens, heads, head_dim, rotary_dim, order, pad, scaling):
    t = torch()
    x = rotary_case(kind, batch, tokens, heads, head_dim, order, pad)
    plan, turns = rotary_plan(rotary_dim, layout, 1.125 if scaling == "banded" else 1.0, scaling)
    far = 1 << 17
    rng = np.random.default_rng(tokens)
    given = rng.integers(-far, far, size=(batch, tokens))
    given[0, 0] = far
    for positions, kind_of in ((given, abi.I64), (given, abi.I32), (given[:1], abi.I64), (None, abi.I32)):
        first = 1000
        if positions is None:
            device, p, stride = None, np.tile(first + np.arange(tokens), (batch, 1)), 0
        else:
            device = t.tensor(positions, device="cuda", dtype=t.int64 if kind_of == abi.I64 else t.int32)
            p = np.broadcast_to(positions, (batch, tokens))
            stride = tokens if len(positions) == batch else 0
        for name, backward in (("geo_b200_rotary", False), ("geo_b200_rotary_vjp", True)):
            y = t.full_like(x, 7.0)
            s = rotary_shape(x, y, position_type=kind_of, position_batch_stride=stride, first_position=first)
            call(name, ctypes.byref(plan), ctypes.byref(s), P(x), P(device), P(y))
            want = ref.rotary(x.double(), p, turns, layout, plan.amplitude, backward)
            ref.assert_within(y, want, ref.rotary_bound(x.double(), want, turns, layout, plan.amplitude, x.dtype, far),
                              name)
            assert t.equal(y[..., rotary_dim:], x[..., rotary_dim:])
        same = t.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda").copy_(x)
        s = rotary_shape(same, same, position_type=kind_of, position_batch_stride=stride, first_position=first)
        call(name, ctypes.byref(plan), ctypes.byref(s), P(same), P(device), P(same))
        assert t.equal(same, y)


@pytest.mark.parametrize("kind", ["f64", "f32"])
def test_rotary_at_the_farthest_positions(kind):
    x = rotary_case(kind, 1, 4, 2, 128)
    positions = np.array([[-(1 << 31), (1 << 31) - 1, 1 << 31, 1234567891]])
    for scaling in ("none", "banded"):
        plan, turns = rotary_plan(128, "half", 1.0, scaling)
        y = torch().empty_like(x)
        call("geo_b200_rotary", ctypes.byref(plan), ctypes.byref(rotary_shape(x, y, position_batch_stride=4)), P(x),
             P(torch().tensor(positions, device="cuda")), P(y))
        want = ref.rotary(x.double(), positions, turns, "half", 1.0)
        ref.assert_within(y, want, ref.rotary_bound(x.double(), want, turns, "half", 1.0, x.dtype, 1 << 31))


def test_rotary_layout_change_and_gaps():
    """From one layout of the heads into another; what lies between the heads stays as it was."""
    t = torch()
    x = rotary_case("bf16", 2, 37, 6, 64)
    whole = t.full((2, 6, 37, 80), 7.0, device="cuda", dtype=x.dtype)
    y = whole[..., 8:72].transpose(1, 2)
    plan, turns = rotary_plan(64, "interleaved")
    call("geo_b200_rotary", ctypes.byref(plan), ctypes.byref(rotary_shape(x, y)), P(x), None, P(y))
    want = t.empty_like(x)
    call("geo_b200_rotary", ctypes.byref(plan), ctypes.byref(rotary_shape(x, want)), P(x), None, P(want))
    assert t.equal(y, want)
    assert (whole[..., :8] == 7).all() and (whole[..., 72:] == 7).all()


def test_rotary_is_a_function_of_the_distance():
    """<R(p) q, R(p + k) v> is the same for every p: 2^-50 of |q| |v| for a few roundings a product."""
    t = torch()
    q, v = rotary_case("f64", 1, 1, 1, 128, seed=1), rotary_case("f64", 1, 1, 1, 128, seed=2)
    plan, _ = rotary_plan(128, "half")
    seen = []
    for p in (0, 1, 77, 100000, 1 << 22):
        turned = []
        for x, at in ((q, p), (v, p + 13)):
            y = t.empty_like(x)
            call("geo_b200_rotary", ctypes.byref(plan), ctypes.byref(rotary_shape(x, y, first_position=at)), P(x), None,
                 P(y))
            turned.append(y)
        seen.append(float((turned[0] * turned[1]).sum()))
    size = float(q.norm() * v.norm())
    assert max(seen) - min(seen) <= 64 * 2.0 ** -52 * size


# ---- streams, graphs, refusals, differences ---------------------------------------


def test_other_stream_and_captured_graph():
    """Forward and VJP in one captured graph: every replay reads the offset that the device holds then, and draws
    what an eager call with that offset draws."""
    t = torch()
    x, res, dy = (make(200, 512, t.bfloat16, seed=s) for s in (1, 2, 3))
    w, b = parameters(512, t.float32)
    n, d = norm_config(x, t.float32), drop_config(x, 0.4, 2, offset=11)
    space, size = workspace(n)
    offset = t.zeros(1, dtype=t.int64, device="cuda")
    out = {k: t.empty_like(x) for k in ("z", "y", "dres", "dx", "drop", "turned")}
    mean, rstd = stats_like(x)
    dw, db = t.empty_like(w), t.empty_like(b)
    plan, _ = rotary_plan(64, "half")
    heads = x.view(1, 200, 8, 64)
    s = rotary_shape(heads, out["turned"].view(1, 200, 8, 64))

    def step(dev_offset, dcfg):
        call("geo_b200_dropout", ctypes.byref(dcfg), P(x), None, dev_offset, P(out["drop"]))
        call("geo_b200_residual_dropout_layer_norm", ctypes.byref(n), ctypes.byref(dcfg), P(x), P(res), dev_offset,
             P(w), P(b), P(out["z"]), P(out["y"]), P(mean), P(rstd))
        call("geo_b200_rotary", ctypes.byref(plan), ctypes.byref(s), P(out["y"]), None, P(out["turned"]))
        call("geo_b200_residual_dropout_layer_norm_vjp", ctypes.byref(n), ctypes.byref(dcfg), dev_offset, P(out["z"]),
             P(w), P(mean), P(rstd), P(dy), P(out["turned"]), P(out["dres"]), P(out["dx"]), P(dw), P(db), P(space),
             size)

    side = t.cuda.Stream()
    side.wait_stream(t.cuda.current_stream())
    graph = t.cuda.CUDAGraph()
    with t.cuda.stream(side):
        step(P(offset), d)
        with t.cuda.graph(graph, stream=side):
            step(P(offset), d)
    t.cuda.synchronize()
    masks = []
    for k in range(3):
        offset.fill_(k)
        graph.replay()
        t.cuda.synchronize()
        got = {name: v.clone() for name, v in out.items()} | {"dw": dw.clone(), "db": db.clone(), "mean": mean.clone()}
        step(None, drop_config(x, 0.4, 2, offset=11 + k))
        for name, v in {**out, "dw": dw, "db": db, "mean": mean}.items():
            assert t.equal(v, got[name]), name
        masks.append(got["drop"] != 0)
    assert not t.equal(masks[0], masks[1]) and not t.equal(masks[1], masks[2])


def test_two_streams_at_once():
    """The same VJP on two streams, each with a workspace of its own, gives the bits of one alone."""
    t = torch()
    x, dy = make(5000, 1024, t.bfloat16, seed=1), make(5000, 1024, t.bfloat16, seed=2)
    w, _ = parameters(1024, t.float32)
    _, mean, rstd = ref.norm(x.double(), None, None, EPS)
    mean, rstd = mean.float(), rstd.float()
    c = norm_config(x, t.float32)
    sets = []
    for _ in range(3):
        space, size = workspace(c)
        sets.append((t.empty_like(x), t.empty_like(w), t.empty_like(w), space, size, t.cuda.Stream()))
    t.cuda.synchronize()
    for dx, dw, db, space, size, side in sets:
        with t.cuda.stream(side):
            for _ in range(5):
                call("geo_b200_layer_norm_vjp", ctypes.byref(c), P(x), P(w), P(mean), P(rstd), P(dy), P(dx), P(dw),
                     P(db), P(space), size)
    t.cuda.synchronize()
    for other in sets[1:]:
        assert all(t.equal(p, q) for p, q in zip(sets[0][:3], other[:3]))


def test_pointer_and_workspace_refusals():
    t = torch()
    L = abi.lib()
    x, host = make(8, 64, t.float32), t.randn(8, 64)
    y, whole = like(x)
    w, b = parameters(64, t.float32)
    mean, rstd = stats_like(x)
    n, d = norm_config(x, t.float32), drop_config(x)
    r, q = ctypes.byref(n), ctypes.byref(d)
    off = ctypes.c_void_p(x.data_ptr() + 2)  # not aligned to a float32
    for bad in (P(host), off):
        assert L.geo_b200_layer_norm(r, bad, P(w), P(b), P(y), None, None, stream()) == INVALID
        assert L.geo_b200_layer_norm(r, P(x), bad, P(b), P(y), None, None, stream()) == INVALID
        assert L.geo_b200_layer_norm(r, P(x), P(w), P(b), P(y), bad, None, stream()) == INVALID
        assert L.geo_b200_dropout(q, bad, None, None, P(y), stream()) == INVALID
        assert L.geo_b200_dropout(q, P(x), bad, None, P(y), stream()) == INVALID
        assert L.geo_b200_dropout(q, P(x), None, bad, P(y), stream()) == INVALID
        assert L.geo_b200_dropout_vjp(q, None, bad, P(y), stream()) == INVALID
    plan, _ = rotary_plan(64, "half")
    heads = x.view(1, 8, 1, 64)
    s = rotary_shape(heads, heads)
    for bad in (P(host), off):
        assert L.geo_b200_rotary(ctypes.byref(plan), ctypes.byref(s), bad, None, P(y), stream()) == INVALID
        assert L.geo_b200_rotary(ctypes.byref(plan), ctypes.byref(s), P(x), bad, P(y), stream()) == INVALID
        assert L.geo_b200_rotary(ctypes.byref(plan), ctypes.byref(s), P(x), None, bad, stream()) == INVALID
    space, size = workspace(n)
    dw, db = t.empty_like(w), t.empty_like(b)

    def vjp(space_pointer, bytes_given):
        return L.geo_b200_layer_norm_vjp(r, P(x), P(w), P(mean), P(rstd), P(x), P(y), P(dw), P(db), space_pointer,
                                         bytes_given, stream())

    assert vjp(None, size) == INVALID
    assert vjp(P(space), size - 1) == INVALID
    assert vjp(ctypes.c_void_p(space.data_ptr() + 8), size) == INVALID
    assert vjp(P(space.cpu()), size) == INVALID
    t.cuda.synchronize()
    assert (whole == 7).all()  # nothing was launched
    pinned = host.pin_memory()  # pinned host memory is reached in place
    assert L.geo_b200_layer_norm(r, P(pinned), P(w), P(b), P(y), None, None, stream()) == 0
    want, _ = like(x)
    call("geo_b200_layer_norm", r, P(pinned.cuda()), P(w), P(b), P(want), None, None)
    assert t.equal(y, want)


def test_fused_equals_its_parts():
    """float64: z of the fused call is dropout's y bit for bit; y is layer norm's of it within the bounds of both."""
    t = torch()
    x, res = make(50, 320, t.float64, seed=1), make(50, 320, t.float64, seed=2)
    w, b = parameters(320, t.float64)
    n, d = norm_config(x, t.float64), drop_config(x, 0.2, 6)
    z, y, z2, y2 = (t.empty_like(x) for _ in range(4))
    call("geo_b200_residual_dropout_layer_norm", ctypes.byref(n), ctypes.byref(d), P(x), P(res), None, P(w), P(b), P(z),
         P(y), None, None)
    call("geo_b200_dropout", ctypes.byref(d), P(x), P(res), None, P(z2))
    call("geo_b200_layer_norm", ctypes.byref(n), P(z2), P(w), P(b), P(y2), None, None)
    assert t.equal(z, z2)
    want = ref.norm(z, w, b, EPS)
    bound = ref.norm_bound(z, w, b, want[2], want[0], t.float64)[0]
    ref.assert_within(y, want[0], bound)
    ref.assert_within(y2, want[0], bound)


def test_layer_of_multivectors_against_differences():
    """The operators as a layer uses them, in float64 on rows of Cl(6,0) multivectors: z, h = the fused call over whole
    multivectors; p = h W (the library's product); r = p turned by its position; loss = <r, c>. The VJPs chained give
    the loss's gradient to x, the residual, weight, bias: against central differences along random directions."""
    t = torch()
    L = abi.lib()
    rows, cols = 24, 64
    x, res, c = (make(rows, cols, t.float64, seed=s) for s in (1, 2, 3))
    w, b = parameters(cols, t.float64)
    par = make(1, cols, t.float64, seed=4, size=0.3).contiguous()
    sig = abi.sig_array((1,) * 6)
    n, d = norm_config(x, t.float64), drop_config(x, 0.25, 6)
    space, size = workspace(n)
    plan, _ = rotary_plan(32, "interleaved", 1.25, "banded")

    def turn(name, v):
        heads, out = v.view(2, rows // 2, 2, 32), t.empty_like(v)
        s = rotary_shape(heads, out.view(2, rows // 2, 2, 32), first_position=4000)
        call(name, ctypes.byref(plan), ctypes.byref(s), P(v), None, P(out))
        return out

    def product(v, m):
        out = t.empty_like(v)
        assert L.geo_b200_forward_f64(6, sig, 0, 0, P(v), P(m), P(out), rows, stream()) == 0
        return out

    def forward(x, res, w, b):
        z, h = t.empty_like(x), t.empty_like(x)
        mean, rstd = stats_like(x)
        call("geo_b200_residual_dropout_layer_norm", ctypes.byref(n), ctypes.byref(d), P(x), P(res), None, P(w), P(b),
             P(z), P(h), P(mean), P(rstd))
        loss = (turn("geo_b200_rotary", product(h, par)) * c).sum() + (z * c).sum()
        return loss, z, mean, rstd

    _, z, mean, rstd = forward(x, res, w, b)
    dp = turn("geo_b200_rotary_vjp", c)
    # The adjoint of multiplication by W is multiplication by its reverse in a Euclidean metric.
    reverse = par.clone()
    for k in range(64):
        if (bin(k).count("1") // 2) % 2:
            reverse[0, k] = -reverse[0, k]
    dh = product(dp, reverse)
    dres, dx, dw, db = t.empty_like(x), t.empty_like(x), t.empty_like(w), t.empty_like(b)
    call("geo_b200_residual_dropout_layer_norm_vjp", ctypes.byref(n), ctypes.byref(d), None, P(z), P(w), P(mean),
         P(rstd), P(dh), P(c), P(dres), P(dx), P(dw), P(db), P(space), size)
    inputs, grads = [x, res, w, b], [dx, dres, dw, db]
    for i, (v, g) in enumerate(zip(inputs, grads)):
        direction = t.randn(v.shape, generator=t.Generator(device="cuda").manual_seed(50 + i), device="cuda",
                            dtype=t.float64)
        step = 1e-5
        losses = []
        for sign in (1, -1):
            moved = list(inputs)
            moved[i] = v + sign * step * direction
            losses.append(float(forward(*moved)[0]))
        slope = (losses[0] - losses[1]) / (2 * step)
        exact = float((g * direction).sum())
        # Differences: 1e-10 of truncation times third derivatives of order one, and 2^-53 |loss| / step.
        size_of = float((g.abs() * direction.abs()).sum())
        assert abs(slope - exact) <= 1e-7 * (size_of + 1), (i, slope, exact)
