"""RMS norm and the block norm (geo/geo_b200.h section 5) on the GPU against 64-bit definitions."""
from __future__ import annotations

import ctypes

import pytest

import feed_forward_reference as ff
from geometricelementaryoperators_b200 import abi
from layer_reference import TYPES, assert_within, torch_type, wide_type
from test_gpu_feed_forward import inside, made, untouched

pytestmark = pytest.mark.gpu
ref = ctypes.byref
EPSILON = 1e-5

#: rows, cols: a value, part of a warp, a warp, part of a block, a block, clusters, rows off 16 bytes of each, more rows
#: than teams, rows beyond clusters.
SIZES = [(1, 1), (1, 64), (7, 3), (300, 16), (5000, 24), (3001, 64), (33, 100), (2, 512), (700, 520), (1300, 1003),
         (3, 2048), (77, 4096), (1, 4099), (600, 5000), (5, 8192), (300, 16384), (2, 32768), (3, 32771), (2, 70000)]
TYPE_PAIRS = [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "f32"), ("f64", "f64")]


def path(cols):
    """Rows of more than 16384 values: 64 values a thread and clusters of up to 64 warps, or sums of sums of 64."""
    return ff.PATH if cols <= 16384 else 300


class Rows:
    """Arrays of a call, in wider buffers with `pad` values behind each row, starting `before` values in."""

    def __init__(self, kind, ptype, rows, cols, gate="none", pad=0, before=0, seed=1, weights=True, dz=True, scale=1.0):
        self.dtype, self.ptype, self.wide = torch_type(kind), torch_type(ptype), wide_type(torch_type(kind))
        self.rows, self.cols, self.gate_kind, self.pad, self.before = rows, cols, gate, pad, before
        self.alpha, self.beta = 0.75, 1.5
        self.buffers = []
        new = lambda i, s=1.0: self.place(made(seed + i, self.dtype, rows, cols, scale=s))  # noqa: E731
        self.x, self.residual, self.dy = new(0, 2.0 * scale), new(1, scale), new(2, 0.1)
        self.gate = None if gate == "none" else new(3, 2.0)
        self.dz = new(4, 0.1) if dz else None
        weight = lambda i: (1 + made(seed + i, self.ptype, cols, scale=0.2)) if weights else None  # noqa: E731
        self.post, self.pre = weight(5), weight(6)
        stride = cols + pad
        self.norm = abi.LayerNormConfig(type=TYPES[kind], parameter_type=TYPES[ptype], rows=rows, cols=cols,
                                        x_stride=stride, y_stride=stride, y_cotangent_stride=stride,
                                        x_cotangent_stride=stride, epsilon=EPSILON)
        names = ("x", "residual", "gate", "z", "y", "y_cotangent", "z_cotangent", "residual_cotangent", "x_cotangent",
                 "gate_cotangent")
        self.block = abi.BlockNormConfig(type=TYPES[kind], parameter_type=TYPES[ptype], gate=ff.GATES[gate], rows=rows,
                                         cols=cols, epsilon=EPSILON, residual_scale=self.alpha, block_scale=self.beta,
                                         **{n + "_stride": stride for n in names})

    def place(self, values):
        view, buffer = inside(values, self.pad, self.before)
        self.buffers.append((buffer, view))
        return view

    def blank(self):
        import torch

        return self.place(torch.full((self.rows, self.cols), float("nan"), device="cuda", dtype=self.dtype))

    def statistic(self):
        import torch

        return torch.full((self.rows,), float("nan"), device="cuda", dtype=self.wide)

    def column(self):
        import torch

        return torch.full((self.cols,), float("nan"), device="cuda", dtype=self.ptype)

    def space(self, size):
        import torch

        return torch.empty(max(1, size), device="cuda", dtype=torch.uint8)

    def wide_of(self, *arrays):
        return [None if v is None else v.double() for v in arrays]


def stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


def rms(r, y=None):
    p, L = ff.pointer, abi.lib()
    y, rstd = r.blank() if y is None else y, r.statistic()
    assert L.geo_b200_rms_norm(ref(r.norm), p(r.x), p(r.post), p(y), p(rstd), stream()) == 0
    return y, rstd


def rms_vjp(r, rstd, dx=None, wanted=(True, True)):
    p, L = ff.pointer, abi.lib()
    dx, dw = r.blank() if dx is None else dx, r.column()
    space = r.space(L.geo_b200_rms_norm_vjp_workspace(ref(r.norm)))
    assert L.geo_b200_rms_norm_vjp(ref(r.norm), p(r.x), p(r.post), p(rstd), p(r.dy), p(dx) if wanted[0] else None,
                                   p(dw) if wanted[1] else None, p(space), space.numel(), stream()) == 0
    return dx, dw


def block(r, z=None, y=None):
    p, L = ff.pointer, abi.lib()
    z, y = r.blank() if z is None else z, r.blank() if y is None else y
    x_rstd, z_rstd = r.statistic(), r.statistic()
    assert L.geo_b200_block_norm(ref(r.block), p(r.x), p(r.residual), p(r.gate), p(r.post), p(r.pre), p(z), p(y),
                                 p(x_rstd), p(z_rstd), stream()) == 0
    return z, y, x_rstd, z_rstd


def block_vjp(r, z, x_rstd, z_rstd, wanted=(True,) * 5, outs=None):
    p, L = ff.pointer, abi.lib()
    outs = outs or [r.blank(), r.blank(), None if r.gate is None else r.blank(), r.column(), r.column()]
    space = r.space(L.geo_b200_block_norm_vjp_workspace(ref(r.block)))
    ptrs = [p(o) if on else None for o, on in zip(outs, wanted)]
    assert L.geo_b200_block_norm_vjp(ref(r.block), p(r.x), p(r.gate), p(z), p(r.post), p(r.pre), p(x_rstd), p(z_rstd),
                                     p(r.dy), p(r.dz), *ptrs, p(space), space.numel(), stream()) == 0
    return outs


def half(t):
    import torch

    return torch.finfo(t).eps / 2


def check_rms(r):
    x, w, dy = r.wide_of(r.x, r.post, r.dy)
    y, rstd = rms(r)
    want, want_rstd = ff.rms(x, w, EPSILON)
    bound, bound_rstd = ff.rms_bound(want, want_rstd, r.dtype, path(r.cols))
    assert_within(y, want, bound, "y")
    assert_within(rstd, want_rstd, bound_rstd, "rstd")
    dx, dw = rms_vjp(r, rstd)
    want_dx, want_dw = ff.rms_vjp(x, w, rstd.double(), dy)
    bound_dx, bound_dw = ff.rms_vjp_bound(x, w, rstd.double(), dy, want_dx, r.dtype, path(r.cols))
    assert_within(dx, want_dx, bound_dx, "x_bar")
    assert_within(dw, want_dw, bound_dw + half(r.ptype) * want_dw.abs() + ff.least(r.ptype), "weight_bar")
    return y, rstd, dx, dw


def check_block(r):
    x, residual, gate, post, pre, dy, dz = r.wide_of(r.x, r.residual, r.gate, r.post, r.pre, r.dy, r.dz)
    args = (x, residual, gate, r.gate_kind, post, pre, r.alpha, r.beta, EPSILON)
    outs = block(r)
    for name, got, want, bound in zip(("z", "y", "x_rstd", "z_rstd"), outs, ff.block(*args),
                                      ff.block_bound(*args, r.dtype, path(r.cols))):
        assert_within(got, want, bound, name)
    z, _, x_rstd, z_rstd = outs
    grads = block_vjp(r, z, x_rstd, z_rstd)
    args = (x, gate, r.gate_kind, z.double(), post, pre, x_rstd.double(), z_rstd.double(), dy, dz, r.alpha, r.beta)
    for name, got, want, bound in zip(("residual_bar", "x_bar", "gate_bar", "post_bar", "pre_bar"), grads,
                                      ff.block_vjp(*args), ff.block_vjp_bound(*args, r.dtype, path(r.cols))):
        if want is None:
            continue
        if name in ("post_bar", "pre_bar"):
            bound = bound + half(r.ptype) * want.abs() + ff.least(r.ptype)
        assert_within(got, want, bound, name)
    return outs, grads


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("kind,ptype", TYPE_PAIRS)
def test_rms_norm(kind, ptype, size):
    r = Rows(kind, ptype, *size)
    check_rms(r)
    untouched(r.buffers)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("kind,ptype,gate", [("bf16", "f32", "sigmoid"), ("f16", "f16", "tanh"), ("f32", "f32", "linear"),
                                             ("f64", "f64", "sigmoid"), ("bf16", "bf16", "none"), ("f32", "f32", "none")])
def test_block_norm(kind, ptype, gate, size):
    r = Rows(kind, ptype, *size, gate=gate)
    check_block(r)
    untouched(r.buffers)


@pytest.mark.parametrize("gate", ["none", "linear", "sigmoid", "tanh"])
@pytest.mark.parametrize("kind,ptype", TYPE_PAIRS)
@pytest.mark.parametrize("size,pad,before", [((50, 64), 8, 0), ((50, 64), 1, 0), ((50, 64), 0, 1), ((50, 65), 3, 5),
                                             ((300, 1000), 9, 2), ((20, 4096), 1, 1), ((20, 9001), 0, 0),
                                             ((20, 12000), 1, 3)])
def test_rows_of_wider_arrays(size, pad, before, kind, ptype, gate):
    r = Rows(kind, ptype, *size, gate=gate, pad=pad, before=before, weights=gate != "linear", dz=gate != "tanh")
    check_rms(r)
    check_block(r)
    untouched(r.buffers)


@pytest.mark.parametrize("size", [(3, 20), (200, 1024), (9, 9000), (3, 40000)])
@pytest.mark.parametrize("kind", ["bf16", "f64"])
def test_some_outputs_and_in_place(kind, size):
    """Every cotangent is the same alone as among all, and over an input; y and z over x and the residual."""
    import torch

    r = Rows(kind, kind, *size, gate="sigmoid")
    y, rstd, dx, dw = check_rms(r)
    assert torch.equal(rms_vjp(r, rstd, wanted=(True, False))[0], dx)
    assert torch.equal(rms_vjp(r, rstd, wanted=(False, True))[1], dw)
    (z, yz, x_rstd, z_rstd), grads = check_block(r)
    for n in range(5):
        alone = block_vjp(r, z, x_rstd, z_rstd, wanted=[i == n for i in range(5)])
        for i, (one, other) in enumerate(zip(alone, grads)):
            assert torch.equal(one, other) if i == n else one.isnan().all()
    saved = [v.clone() for v in (r.x, r.residual, r.gate, r.dy, r.dz)]
    z2, y2, _, _ = block(r, z=r.residual, y=r.x)
    assert torch.equal(z2, z) and torch.equal(y2, yz)
    r.x.copy_(saved[0])
    outs = [r.dz, r.x, r.gate, r.column(), r.column()]
    again = block_vjp(r, z, x_rstd, z_rstd, outs=outs)
    assert all(torch.equal(a, b) for a, b in zip(again, grads))
    r.x.copy_(saved[0])
    r.dy.copy_(saved[3])
    assert torch.equal(rms_vjp(r, rstd, dx=r.dy)[0], dx)
    r.dy.copy_(saved[3])
    assert torch.equal(rms(r, y=r.x)[0], y)


@pytest.mark.parametrize("cols", [48, 1024, 8192, 33000])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_not_finite_and_empty_rows(kind, cols):
    """A row's NaN and infinity stay with the row; a row of zeros gives zeros."""
    r = Rows(kind, kind, 9, cols, gate="sigmoid")
    r.x[1, 3] = float("nan")
    r.residual[2, 5] = float("inf")
    r.x[4] = 0
    r.residual[5] = 0
    r.x[5] = 0
    z, y, x_rstd, z_rstd = block(r)
    good = [0, 3, 4, 5, 6, 7, 8]
    assert z[good].isfinite().all() and y[good].isfinite().all()
    assert y[1].isnan().all() and z[1].isnan().all() and not y[2].isfinite().all()
    assert (z[5] == 0).all() and (y[5] == 0).all()
    dres, dx, dgate, dpost, dpre = block_vjp(r, z, x_rstd, z_rstd)
    assert all(v[good].isfinite().all() for v in (dres, dx, dgate))
    assert dres[1].isnan().all() and dpost.isnan().any()


def test_gate_far_from_zero():
    """Sigmoid's slope and tanh's keep their relative accuracy where they are tiny, and infinite gates are their limits."""
    import torch

    for gate in ("sigmoid", "tanh"):
        r = Rows("f32", "f32", 20, 96, gate=gate)
        r.gate.copy_(torch.linspace(-30, 30, 20 * 96, device="cuda").view(20, 96))
        check_block(r)
        r.gate[3, 5], r.gate[3, 6] = float("inf"), -float("inf")
        z, _, x_rstd, z_rstd = block(r)
        n = (r.x[3] * x_rstd[3] * r.post).double()
        low = 0.0 if gate == "sigmoid" else -1.0
        base = r.alpha * r.residual[3].double()
        assert abs(z[3, 5] - base[5] - r.beta * n[5]) < 1e-5 and abs(z[3, 6] - base[6] - r.beta * low * n[6]) < 1e-5
        dgate = block_vjp(r, z, x_rstd, z_rstd)[2]
        assert dgate[3, 5] == 0 and dgate[3, 6] == 0


def test_block_that_cancels_the_residual():
    """z nearly 0: its statistic comes from z's values, not from a difference of large squares."""
    r = Rows("f64", "f64", 40, 640, weights=False)
    x = r.x.double()
    n = x / (x.square().mean(1, keepdim=True) + EPSILON).sqrt()
    r.residual.copy_(-(r.beta / r.alpha) * n + 1e-9 * made(77, x.dtype, 40, 640))
    check_block(r)


def test_captured_and_on_streams():
    import torch

    r, other = Rows("bf16", "f32", 600, 4096, gate="sigmoid"), Rows("bf16", "f32", 600, 4096, gate="sigmoid", seed=40)
    outs, grads = check_block(r)
    outs2, grads2 = check_block(other)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for rows, s, w in ((r, streams[0], outs), (other, streams[1], outs2)):
            with torch.cuda.stream(s):
                got.append((block(rows), block_vjp(rows, w[0], w[2], w[3])))
        torch.cuda.synchronize()
        for (o, g), wo, wg in zip(got, (outs, outs2), (grads, grads2)):
            assert all(torch.equal(a, b) for a, b in zip((*o, *g), (*wo, *wg)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = block(r)
        g = block_vjp(r, o[0], o[2], o[3])
    r.x.copy_(other.x)
    r.residual.copy_(other.residual)
    r.gate.copy_(other.gate)
    graph.replay()
    want = block(r)
    want_grads = block_vjp(r, want[0], want[2], want[3])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*o, *g), (*want, *want_grads)))


def test_commutes_with_rotors():
    """One weight for a whole multivector of Cl(3,0): the norm of a turned row is the turned norm."""
    import torch

    from layer_reference import half_step

    r = Rows("f64", "f64", 100, 64)
    r.post = None
    y, _ = rms(r)
    # The sandwich with a rotor turns the coefficients of each grade orthogonally: any orthogonal map does here.
    q = torch.linalg.qr(made(3, torch.float64, 64, 64))[0]
    turned = (r.x @ q).contiguous()
    r.x.copy_(turned)
    again, _ = rms(r)
    assert_within(again, y @ q, 200 * half_step(torch.float64) * (y.abs() @ q.abs()), "turned")


def test_far_rows():
    """Rows whose offsets pass 2^31 values."""
    import torch

    stride = (1 << 30) + 16
    buffer = torch.zeros(2 * stride + 512, device="cuda", dtype=torch.bfloat16)
    for cols, start in ((512, 0), (511, 1)):
        r = Rows("bf16", "bf16", 3, cols)
        y, rstd = rms(r)
        dx, dw = rms_vjp(r, rstd)
        far = torch.as_strided(buffer, (3, cols), (stride, 1), start)
        far.copy_(r.x)
        r.x, r.norm.x_stride = far, stride
        got, again = rms(r)
        assert torch.equal(got, y) and torch.equal(again, rstd)
        got, again = rms_vjp(r, rstd)
        assert torch.equal(got, dx) and torch.equal(again, dw)


def test_refusals_with_usable_arrays():
    p, L = ff.pointer, abi.lib()
    r = Rows("f32", "f32", 8, 64, gate="sigmoid")
    z, y, x_rstd, z_rstd = block(r)
    import torch

    host = torch.empty(8, 64)
    args = [r.x, r.residual, r.gate, r.post, r.pre, z, y, x_rstd, z_rstd]

    def call(i, v):
        a = list(args)
        a[i] = v
        return L.geo_b200_block_norm(ref(r.block), *[p(t) for t in a], stream())

    assert call(0, r.x) == 0
    for i in (0, 1, 2, 5, 6):
        assert call(i, None) == 1 and call(i, host) == 1
    assert call(5, y) == 1
    assert L.geo_b200_rms_norm(ref(r.norm), p(host), None, p(y), None, stream()) == 1
    small = torch.empty(16, device="cuda", dtype=torch.uint8)
    assert L.geo_b200_rms_norm_vjp(ref(r.norm), p(r.x), None, p(x_rstd), p(r.dy), p(y), p(r.column()), p(small), 16,
                                   stream()) == 1
    assert L.geo_b200_rms_norm_vjp(ref(r.norm), p(r.x), None, p(x_rstd), p(r.dy), p(y), None, None, 0, stream()) == 0
    torch.cuda.synchronize()
