"""Gated feed-forward block (geo/geo_b200.h section 5) on the GPU against 64-bit definitions."""
from __future__ import annotations

import ctypes

import pytest

import feed_forward_reference as ff
from geometricelementaryoperators_b200 import abi
from layer_reference import TYPES, assert_within, torch_type

pytestmark = pytest.mark.gpu
ref = ctypes.byref

#: rows, cols, hidden: one value, a token, few rows, one row past a kernel's limits, ragged tiles, several tiles a
#: multiprocessor, results too small for every multiprocessor with many rows (their sums cut into parts).
SIZES = [(1, 1, 1), (1, 64, 256), (2, 1000, 333), (4, 1003, 77), (5, 8, 1000), (8, 256, 264), (9, 65, 130),
         (17, 72, 40), (100, 33, 65), (127, 128, 256), (129, 136, 264), (300, 520, 1032), (2600, 72, 200),
         (5000, 64, 64), (1500, 1400, 2072)]


def made(seed, dtype, *shape, scale=1.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float64) * scale).to(dtype)


def inside(values, pad=0, before=0, fill=7.0):
    """The values as rows of a wider buffer, `before` values from its start on, `pad` behind each row; what lies
    around them is `fill`. The buffer comes with them."""
    import torch

    rows, cols = values.shape
    buffer = torch.full((before + rows * (cols + pad),), fill, device="cuda", dtype=values.dtype)
    view = buffer[before:].view(rows, cols + pad)[:, :cols]
    view.copy_(values)
    return view, buffer


class Case:
    """Inputs, the library's outputs for them, and what they are to be."""

    def __init__(self, kind, rows, cols, hidden, activation="silu", gradient=None, pad=0, before=0, weight_pad=0, seed=1,
                 scale=1.0):
        import torch

        self.dtype, self.activation = torch_type(kind), activation
        self.gradient = torch_type(gradient) if gradient else self.dtype
        self.rows, self.cols, self.hidden, self.pad, self.before = rows, cols, hidden, pad, before
        place = lambda v, p=pad: inside(v, p, before)  # noqa: E731
        self.x, self.x_buffer = place(made(seed, self.dtype, rows, cols, scale=scale))
        self.wg = place(made(seed + 1, self.dtype, hidden, cols, scale=cols ** -0.5), weight_pad)[0]
        self.wu = place(made(seed + 2, self.dtype, hidden, cols, scale=cols ** -0.5), weight_pad)[0]
        self.wd = place(made(seed + 3, self.dtype, cols, hidden, scale=hidden ** -0.5), weight_pad)[0]
        self.dy = place(made(seed + 4, self.dtype, rows, cols))[0]
        self.config = abi.FeedForwardConfig(
            type=TYPES[kind], gradient_type=TYPES[gradient or kind], activation=ff.ACTIVATIONS[activation], rows=rows,
            cols=cols, hidden=hidden, x_stride=cols + pad, y_stride=cols + pad, y_cotangent_stride=cols + pad,
            x_cotangent_stride=cols + pad, gate_weight_stride=cols + weight_pad, up_weight_stride=cols + weight_pad,
            down_weight_stride=hidden + weight_pad, gate_stride=hidden + pad, up_stride=hidden + pad)
        L = abi.lib()
        self.space = torch.empty(L.geo_b200_feed_forward_workspace(ref(self.config)), device="cuda", dtype=torch.uint8)
        self.vjp_space = torch.empty(L.geo_b200_feed_forward_vjp_workspace(ref(self.config)), device="cuda",
                                     dtype=torch.uint8)

    def blank(self, rows, cols, pad, dtype=None):
        import torch

        return inside(torch.full((rows, cols), float("nan"), device="cuda", dtype=dtype or self.dtype), pad, self.before)

    def forward(self, save=True, stream=None):
        import torch

        p = ff.pointer
        y, y_buffer = self.blank(self.rows, self.cols, self.pad)
        a = u = None
        buffers = [(y_buffer, y)]
        if save:
            a, b = self.blank(self.rows, self.hidden, self.pad)
            u, c = self.blank(self.rows, self.hidden, self.pad)
            buffers += [(b, a), (c, u)]
        status = abi.lib().geo_b200_feed_forward(
            ref(self.config), p(self.x), p(self.wg), p(self.wu), p(self.wd), p(a), p(u), p(y), p(self.space),
            self.space.numel(), stream if stream is not None else torch.cuda.current_stream().cuda_stream)
        assert status == 0
        return a, u, y, buffers

    def vjp(self, a, u, stream=None, wanted=(True,) * 4):
        import torch

        p = ff.pointer
        w = self.config.gate_weight_stride - self.cols
        outs = [self.blank(self.rows, self.cols, self.pad), self.blank(self.hidden, self.cols, w, self.gradient),
                self.blank(self.hidden, self.cols, w, self.gradient), self.blank(self.cols, self.hidden, w, self.gradient)]
        ptrs = [p(o[0]) if on else None for o, on in zip(outs, wanted)]
        status = abi.lib().geo_b200_feed_forward_vjp(
            ref(self.config), p(self.x), p(self.wg), p(self.wu), p(self.wd), p(a), p(u), p(self.dy), *ptrs,
            p(self.vjp_space), self.vjp_space.numel(),
            stream if stream is not None else torch.cuda.current_stream().cuda_stream)
        assert status == 0
        return [o[0] for o in outs], [(o[1], o[0]) for o in outs]

    def wide(self):
        return [v.double() for v in (self.x, self.wg, self.wu, self.wd)]

    def check_forward(self, a, u, y):
        want = ff.forward(*self.wide(), self.activation)
        bound = ff.forward_bound(*self.wide(), self.activation, self.dtype)
        for name, got, w, b in zip(("gate", "up", "y"), (a, u, y), want, bound):
            if got is not None:
                assert_within(got, w, b, name)

    def check_vjp(self, a, u, outs, wanted=(True,) * 4):
        args = (*self.wide(), a.double(), u.double(), self.dy.double(), self.activation)
        want = ff.vjp(*args)
        bound = ff.vjp_bound(*args, self.dtype, self.gradient)
        for name, got, w, b, on in zip(("x_bar", "gate_weight_bar", "up_weight_bar", "down_weight_bar"), outs, want,
                                       bound, wanted):
            if on:
                assert_within(got, w, b, name)
            else:
                assert got.isnan().all(), name


def untouched(buffers, fill=7.0):
    """Nothing around the rows was written."""
    for buffer, view in buffers:
        around = buffer.clone()
        around[buffer.numel() - view.shape[0] * view.stride(0):].view(view.shape[0], view.stride(0))[
            :, :view.shape[1]] = fill
        assert (around == fill).all()


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("kind,activation", [("bf16", "silu"), ("f16", "gelu"), ("f32", "sigmoid"), ("f64", "relu")])
def test_block(kind, activation, size):
    c = Case(kind, *size, activation)
    a, u, y, buffers = c.forward()
    c.check_forward(a, u, y)
    outs, more = c.vjp(a, u)
    c.check_vjp(a, u, outs)
    untouched(buffers + more)


@pytest.mark.parametrize("activation", list(ff.ACTIVATIONS))
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32", "f64"])
def test_activations(kind, activation):
    """Wide arguments: gate values of several tens."""
    c = Case(kind, 70, 64, 96, activation, scale=12.0)
    a, u, y, _ = c.forward()
    c.check_forward(a, u, y)
    c.check_vjp(a, u, c.vjp(a, u)[0])


@pytest.mark.parametrize("size", [(1, 64, 128), (3, 65, 30), (40, 65, 130), (300, 136, 264), (3000, 24, 40)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_float32_cotangents_of_weights(kind, size):
    """Their bound is float32's: the inner values come as the sum of two 16-bit ones."""
    c = Case(kind, *size, "silu", gradient="f32")
    a, u, _, _ = c.forward()
    outs, buffers = c.vjp(a, u)
    c.check_vjp(a, u, outs)
    untouched(buffers)


@pytest.mark.parametrize("size", [(3, 64, 72), (9, 64, 72), (40, 65, 130), (200, 136, 264)])
@pytest.mark.parametrize("pad,before,weight_pad", [(8, 8, 8), (8, 0, 1), (1, 0, 0), (3, 0, 5), (0, 1, 0), (8, 3, 8)])
@pytest.mark.parametrize("kind,gradient", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "f32"),
                                           ("f64", "f64")])
def test_rows_of_wider_arrays(kind, gradient, pad, before, weight_pad, size):
    """Strides on and off 16 bytes, and starts off 16 bytes."""
    c = Case(kind, *size, "gelu", gradient=gradient, pad=pad, before=before, weight_pad=weight_pad)
    a, u, y, buffers = c.forward()
    c.check_forward(a, u, y)
    outs, more = c.vjp(a, u)
    c.check_vjp(a, u, outs)
    untouched(buffers + more)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [3, 200])
def test_forward_alone_and_some_cotangents(kind, rows):
    """y is the same with and without the saved projections; each cotangent the same alone as among all."""
    import torch

    c = Case(kind, rows, 72, 136, gradient="f32")
    a, u, y, _ = c.forward()
    assert torch.equal(c.forward(save=False)[2], y)
    outs, _ = c.vjp(a, u)
    c.check_vjp(a, u, outs)
    for wanted in [(True, False, False, False), (False, True, False, False), (False, False, True, False),
                   (False, False, False, True), (True, False, True, True)]:
        again, _ = c.vjp(a, u, wanted=wanted)
        for on, one, other in zip(wanted, again, outs):
            assert torch.equal(one, other) if on else one.isnan().all()


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32", "f64"])
@pytest.mark.parametrize("rows", [4, 150])
def test_not_finite(kind, rows):
    """A row with a NaN, one with an infinity: theirs are the only rows of the outputs that are not finite, and all
    the weights' cotangents that they enter are."""
    c = Case(kind, rows, 64, 72)
    c.x[1, 5] = float("nan")
    c.x[2, 7] = float("inf")
    a, u, y, _ = c.forward()
    bad = [1, 2]
    good = [r for r in range(rows) if r not in bad]
    for v in (a, u, y):
        assert v[good].isfinite().all()
        assert (~v[bad].isfinite()).all(dim=1).all()
    (dx, dwg, dwu, dwd), _ = c.vjp(a, u)
    assert dx[good].isfinite().all() and (~dx[1].isfinite()).all()
    for w in (dwg, dwu, dwd):
        assert (~w.isfinite()).any()


@pytest.mark.parametrize("kind,size", [("bf16", (300, 200, 136)), ("f16", (2, 200, 136)), ("f64", (3000, 40, 24))])
def test_same_bits_captured_and_on_streams(kind, size):
    """The same call twice, in a replayed graph, and on two streams at once with a workspace each."""
    import torch

    c, other = Case(kind, *size), Case(kind, *size, seed=9)
    first, second = c.forward(), other.forward()
    grads, more = c.vjp(*first[:2])[0], other.vjp(*second[:2])[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = [s.forward(stream=t.cuda_stream) + (s.vjp(*w[:2], stream=t.cuda_stream)[0],)
               for s, t, w in ((c, streams[0], first), (other, streams[1], second))]
        torch.cuda.synchronize()
        for g, w, d in zip(got, (first, second), (grads, more)):
            assert torch.equal(g[2], w[2])
            assert all(torch.equal(p, q) for p, q in zip(g[4], d))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, u, y, _ = c.forward()
        outs, _ = c.vjp(a, u)
    c.x.copy_(other.x)
    graph.replay()
    want = c.forward()
    want_grads, _ = c.vjp(*want[:2])
    torch.cuda.synchronize()
    assert torch.equal(y, want[2]) and not torch.equal(y, first[2])
    assert all(torch.equal(p, q) for p, q in zip(outs, want_grads))


@pytest.mark.parametrize("kind", ["f64", "f32"])
def test_against_differences(kind):
    """y_bar . (y(x + d) - y(x - d)) / 2 = x_bar . d, and so for the weights. Central differences in float64 are off by
    the third derivative, (10^-4)^2 of the slope, and by rounding, 10^-16 / 10^-4; float32's own VJP by its bound."""
    import torch

    c = Case(kind, 12, 16, 24, "silu")
    a, u, _, _ = c.forward()
    outs, _ = c.vjp(a, u)
    args = c.wide()
    for i, got in enumerate(outs):
        d = made(50 + i, torch.float64, *args[i].shape)
        at = lambda h: ff.forward(*[v + h * d if n == i else v for n, v in enumerate(args)], "silu")[2]  # noqa: E731
        slope = ((at(1e-4) - at(-1e-4)) / 2e-4 * c.dy.double()).sum()
        along = (got.double() * d).sum()
        size = (got.double() * d).abs().sum()
        assert abs(slope - along) <= size * (1e-6 if kind == "f64" else 1e-4)


def test_far_rows():
    """Rows whose offsets pass 2^31 values."""
    import torch

    for rows, stride in ((3, (1 << 30) + 8), (9, (1 << 28) + 8)):  # few rows; the tensor cores' kernels
        c = Case("bf16", rows, 64, 72)
        want = c.forward()[2]
        buffer = torch.empty((rows - 1) * stride + 64, device="cuda", dtype=torch.bfloat16)
        far = torch.as_strided(buffer, (rows, 64), (stride, 1))
        far.copy_(c.x)
        c.x, c.config.x_stride = far, stride
        assert torch.equal(c.forward()[2], want)


def test_refusals_with_usable_arrays():
    """What the documentation refuses, with arrays that are good otherwise."""
    import torch

    p, L = ff.pointer, abi.lib()
    c = Case("bf16", 16, 64, 72)
    a, u, y, _ = c.forward()
    stream = torch.cuda.current_stream().cuda_stream

    def call(x=c.x, wg=c.wg, gate=a, up=u, out=y, space=c.space, size=None):
        return L.geo_b200_feed_forward(ref(c.config), p(x), p(wg), p(c.wu), p(c.wd), p(gate), p(up), p(out), p(space),
                                       space.numel() if size is None else size, stream)

    assert call() == 0
    assert call(x=None) == 1 and call(wg=None) == 1 and call(out=None) == 1 and call(gate=None) == 1
    assert call(out=c.x) == 1 and call(gate=u) == 1 and call(size=c.space.numel() - 1) == 1
    assert call(x=torch.empty(16, 64, dtype=torch.bfloat16)) == 1  # pageable host memory
    odd = torch.empty(c.space.numel() + 256, device="cuda", dtype=torch.uint8)[1:]
    assert call(space=odd) == 1
    host = torch.empty(16, 64, dtype=torch.bfloat16).pin_memory()
    host.copy_(c.x)
    assert call(x=host) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows,cols,hidden,block", [(40, 640, 520, 0), (40, 640, 520, 2), (300, 640, 520, 0),
                                                    (700, 640, 520, 3), (5000, 256, 2048, 0), (5000, 256, 2048, 3)])
def test_waits_give_up(rows, cols, hidden, block):
    """Copies that stop (single blocks, parts of K, pairs of blocks), before any tile is whole: the call ends, what they
    were for is NaN, and the next call is right."""
    import torch

    p, L = ff.pointer, abi.lib()
    c = Case("bf16", rows, cols, hidden)
    a, u, y, _ = c.forward()
    args = (ref(c.config), p(c.x), p(c.wg), p(c.wu), p(c.wd))
    (ga, _), (gu, _), (gy, _) = (c.blank(rows, n, 0) for n in (hidden, hidden, cols))
    stream = torch.cuda.current_stream().cuda_stream
    for limit in (1 << 8, 1 << 12):
        assert L.geo_b200_feed_forward_wait_selftest(*args, p(ga), p(gu), p(gy), p(c.space), c.space.numel(), block,
                                                     limit, stream) == 0
        torch.cuda.synchronize()
        assert ga.isnan().all() and gu.isnan().all() and gy.isnan().all()
    for bad in (0, (1 << 20) + 1):
        assert L.geo_b200_feed_forward_wait_selftest(*args, p(ga), p(gu), p(gy), p(c.space), c.space.numel(), 0, bad,
                                                     stream) == 1
    again = c.forward()
    assert all(torch.equal(v, w) for v, w in zip(again[:3], (a, u, y)))
    # A call that other kernels take has no such waits.
    few = Case("bf16", 1, cols, hidden)
    assert L.geo_b200_feed_forward_wait_selftest(ref(few.config), p(few.x), p(few.wg), p(few.wu), p(few.wd), None, None,
                                                 p(gy), p(few.space), few.space.numel(), 0, 16, stream) == 1


def test_host_threads():
    """Calls of several host threads at once, each on a stream and with a workspace of its own, of sizes that take other
    kernels and other amounts of shared memory."""
    import threading

    import torch

    cases = [Case("bf16", 300, 200, 136), Case("bf16", 40, 640, 520, gradient="f32"), Case("f64", 70, 33, 65),
             Case("f32", 200, 136, 264), Case("f16", 2, 1000, 333)]
    want = []
    for c in cases:
        a, u, y, _ = c.forward()
        want.append((a, u, y, c.vjp(a, u)[0]))
    torch.cuda.synchronize()
    failed = []

    def work(c, w):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                a, u, y, _ = c.forward()
                grads, _ = c.vjp(w[0], w[1])
                s.synchronize()
                same = [torch.equal(p, q) for p, q in zip((a, u, y, *grads), (*w[:3], *w[3]))]
                if not all(same):
                    failed.append((c.rows, same))

    threads = [threading.Thread(target=work, args=p) for p in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.parametrize("kind,size", [("bf16", (200000, 40, 24)), ("f16", (3, 131072, 16)), ("bf16", (40, 8, 131072)),
                                       ("f32", (1, 16, 1048576)), ("f64", (130, 100000, 24)), ("f32", (200000, 40, 24))])
def test_long_and_wide(kind, size):
    c = Case(kind, *size, "silu", gradient="f32" if kind == "bf16" else None)
    a, u, y, buffers = c.forward()
    c.check_forward(a, u, y)
    outs, more = c.vjp(a, u)
    c.check_vjp(a, u, outs)
    untouched(buffers + more)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_float32_cotangents_over_many_rows(kind):
    """Their 2-norm's error does not grow with the rows: two terms leave 2^-18 of an inner value (bfloat16; and float16's
    least, 2^-25 of values of some 2^-5), each of the 64 instructions of 16 that sum h_bar's parts, and each of the 128
    that sum a cotangent's, may cut one unit, 2^-23, off a sum's size. Random signs keep the sums of parts to that."""
    c = Case(kind, 8192, 512, 256, gradient="f32")
    a, u, _, _ = c.forward()
    outs, _ = c.vjp(a, u)
    want = ff.vjp(*c.wide(), a.double(), u.double(), c.dy.double(), "silu")
    for got, w in zip(outs[1:], want[1:]):
        assert (got.double() - w).norm() <= (2.0 ** -18 + 192 * 2.0 ** -23) * w.norm()
