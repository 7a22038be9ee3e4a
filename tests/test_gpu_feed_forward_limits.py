"""Gated feed-forward block (geo/geo_b200.h section 5) at its limits on the GPU: waits that give up anywhere, float16
values at both ends of its range, sums of very many values."""
from __future__ import annotations

import ctypes

import pytest

import feed_forward_reference as ff
from geometricelementaryoperators_b200 import abi
from test_gpu_feed_forward import Case

pytestmark = pytest.mark.gpu
ref = ctypes.byref


@pytest.mark.parametrize("rows,cols,hidden", [(40, 640, 520), (300, 640, 520), (5000, 256, 2048), (1100, 2000, 4104)])
def test_any_wait_gives_up(rows, cols, hidden):
    """Waits that look so seldom that any of them may give up, whichever warp's and whichever block's of a pair, with
    copies that stop early, late or not at all: the call ends, every value is NaN or what it is otherwise, and the
    next call is right."""
    import torch

    p, L = ff.pointer, abi.lib()
    c = Case("bf16", rows, cols, hidden)
    want = c.forward()[:3]
    stream = torch.cuda.current_stream().cuda_stream
    for limit in (1, 2, 5, 40):
        for block in (0, 7, 40, 0xFFFFFFFF):
            (a, _), (u, _), (y, _) = (c.blank(rows, n, 0) for n in (hidden, hidden, cols))
            assert L.geo_b200_feed_forward_wait_selftest(
                ref(c.config), p(c.x), p(c.wg), p(c.wu), p(c.wd), p(a), p(u), p(y), p(c.space), c.space.numel(), block,
                limit, stream) == 0
            torch.cuda.synchronize()
            for got, w in zip((a, u, y), want):
                assert ((got == w) | got.isnan()).all()
    assert all(torch.equal(v, w) for v, w in zip(c.forward()[:3], want))


def off(got, want):
    """2-norm of the difference and of what it is of."""
    return float((got.double() - want).norm()), float(want.norm())


@pytest.mark.parametrize("size", [(3, 256, 136), (300, 520, 1032), (4000, 256, 136)])
@pytest.mark.parametrize("before", [0, 1])  # on the tensor cores, and value by value
@pytest.mark.parametrize("gradient", ["f32", "f16"])
@pytest.mark.parametrize("scale", [1e-2, 1e-4, 1e-6])
def test_small_float16_cotangents(gradient, scale, before, size):
    """y_bar as small as a mean over many values makes it. Inner values are multiplied into float16's range, so that
    they are one rounding off, 2^-11, or two terms' 2^-22 on their way to a float32 cotangent of weights; up to 64
    instructions of 16 cut a unit, 2^-23, of a part of h_bar's and a cotangent's sums each, float32's functions leave
    2^-20, and a float16 result has its own rounding, 2^-11 of it or 2^-25."""
    c = Case("f16", *size, "silu", gradient=None if gradient == "f16" else gradient, before=before)
    a, u, _, _ = c.forward()
    c.dy.mul_(scale)
    outs, _ = c.vjp(a, u)
    want = ff.vjp(*c.wide(), a.double(), u.double(), c.dy.double(), "silu")
    sums = 128 * 2.0 ** -23 + 2.0 ** -20
    for n, (got, w) in enumerate(zip(outs, want)):
        difference, of = off(got, w)
        if n == 0 or gradient == "f16":
            assert difference <= (2 * 2.0 ** -11 + sums) * of + 2.0 ** -25 * w.numel() ** 0.5, n
        else:
            assert difference <= (2.0 ** -22 + sums) * of, n


@pytest.mark.parametrize("before", [0, 1])
def test_float16_cotangents_with_infinite_rows(before):
    """A row whose cotangent is not finite leaves the other rows' x_bar as exact as it is without it."""
    c = Case("f16", 300, 256, 136, before=before)
    a, u, _, _ = c.forward()
    c.dy.mul_(1e-6)
    want = ff.vjp(*c.wide(), a.double(), u.double(), c.dy.double(), "silu")[0]
    c.dy[7, 5], c.dy[80, 0] = float("inf"), float("nan")
    got = c.vjp(a, u)[0][0]
    good = [r for r in range(300) if r not in (7, 80)]
    assert (~got[[7, 80]].isfinite()).any(dim=1).all()
    difference, of = off(got[good], want[good])
    assert difference <= (2 * 2.0 ** -11 + 2.0 ** -16) * of + 2.0 ** -25 * want.numel() ** 0.5


@pytest.mark.parametrize("size", [(3, 256, 3000), (300, 256, 136), (300, 1000, 4001), (5000, 24, 40), (2000, 33, 200)])
@pytest.mark.parametrize("before", [0, 1])
def test_float16_rows_of_unlike_sizes(before, size):
    """One row's cotangent and another's projections far above all others: the other rows' x_bar has its digits, as in
    the test of small cotangents."""
    import torch

    c = Case("f16", *size, before=before)
    a, u, _, _ = c.forward()
    c.dy[0] *= 3000.0
    u[1, ::7] *= 4000.0
    want = ff.vjp(*c.wide(), a.double(), u.double(), c.dy.double(), "silu")[0]
    got = c.vjp(a, u)[0][0]
    difference, of = off(got[2:], want[2:])
    assert difference <= (2 * 2.0 ** -11 + 2.0 ** -16) * of + 2.0 ** -25 * want.numel() ** 0.5


@pytest.mark.parametrize("gradient", ["f32", "f16"])
@pytest.mark.parametrize("before", [0, 1])
def test_float16_h_beyond_its_range(gradient, before):
    """act(gate) up of up to 250000 in the VJP: down_weight's cotangent is finite and right."""
    import torch

    c = Case("f16", 200, 64, 72, gradient=None if gradient == "f16" else gradient, before=before)
    a, u = (torch.rand(200, 72, device="cuda").mul(250).add(250).half() for _ in range(2))
    c.dy.mul_(2.0 ** -14)
    got = c.vjp(a, u)[0]
    want = ff.vjp(*c.wide(), a.double(), u.double(), c.dy.double(), "silu")
    for n, (g, w) in enumerate(zip(got, want)):
        difference, of = off(g, w)
        assert difference <= (2 * 2.0 ** -11 + 2.0 ** -16) * of + 2.0 ** -25 * w.numel() ** 0.5, n


@pytest.mark.parametrize("rows,cols,hidden", [(40, 1 << 20, 16), (40, 16, 1 << 20), (1 << 22, 16, 24)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_long_sums_of_like_signs(kind, rows, cols, hidden):
    """Positive values alone, the worst for sums that are cut where others are rounded: what the cuts of one product
    take off is to stay below a quarter of a step of the type's own rounding, and below 2^-12. Two such products follow
    one another, or three in the VJP, and 16-bit values between them and at the end add a rounding each."""
    import torch

    c = Case(kind, rows, cols, hidden, "relu")
    for v, size in ((c.x, 1.0), (c.wg, 4.0 / cols), (c.wu, 4.0 / cols), (c.wd, 4.0 / hidden), (c.dy, 16.0 / rows)):
        v.copy_(torch.rand(v.shape, device="cuda").add(1.0).mul(size))
    t = torch.finfo(c.dtype).eps / 2
    cut = min(t / 2, 2.0 ** -12)
    a, u, y, _ = c.forward()
    want = ff.forward(*c.wide(), "relu")
    for n, (got, w) in enumerate(zip((a, u, y), want)):
        far = ((got.double() - w) / w).abs().max()
        assert far <= (3 * cut + 2 * t if n == 2 else cut + t) * 1.01, n
    outs, _ = c.vjp(a, u)
    want = ff.vjp(*c.wide(), a.double(), u.double(), c.dy.double(), "relu")
    for n, (got, w) in enumerate(zip(outs, want)):
        over = w > 1.1 * torch.finfo(c.dtype).max  # float16's weights' cotangents where cols are many
        assert got[over].isinf().all(), n
        far = ((got.double() - w) / w)[~over].abs()
        assert (far <= ((2 * cut if n < 3 else cut) + 2 * t) * 1.01).all(), n


@pytest.mark.parametrize("kind,size", [("bf16", (200000, 40, 24)), ("f16", (200000, 40, 24)), ("f16", (3, 131072, 16)),
                                       ("bf16", (40, 8, 131072)), ("f32", (1, 16, 1 << 20)), ("f32", (200000, 40, 24)),
                                       ("f64", (130, 100000, 24)), ("bf16", (2, 1 << 18, 40)), ("f32", (70, 200000, 24))])
@pytest.mark.parametrize("gradient", ["f32", None])
def test_long_sums_as_a_whole(kind, gradient, size):
    """2-norms, which sums that leave anything out do not meet: a 64th of K is an eighth of a sum of random signs. 16-bit
    results are two roundings off, twice half a step, the sums' own errors far below; float32 ones sqrt(K) u of rounding
    (2^-14 at 2^20) or two 16-bit terms' 2^-18 and cut parts of 64 instructions, 2^-16: 2^-12 is above all of them and
    their functions; float64 ones sqrt(K) 2^-53."""
    import torch

    if kind == "f64" and gradient:
        pytest.skip("no such pair of types")
    c = Case(kind, *size, "silu", gradient=gradient)
    limit = {torch.float64: 2.0 ** -40, torch.float32: 2.0 ** -12, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
    a, u, y, _ = c.forward()
    want = ff.forward(*c.wide(), "silu")
    for n, (got, w) in enumerate(zip((a, u, y), want)):
        difference, of = off(got, w)
        assert difference <= limit[got.dtype] * of, n
    outs, _ = c.vjp(a, u)
    args = (a.double(), u.double(), c.dy.double(), "silu")
    want = ff.vjp(*c.wide(), *args)
    for n, (got, w) in enumerate(zip(outs, want)):
        difference, of = off(got, w)
        assert difference <= limit[got.dtype] * of, n
    # The check sees what a part of the rows leaves out of the weights' cotangents, or of hidden values out of x_bar.
    rows, hidden = size[0] - (size[0] + 63) // 64, size[2] - (size[2] + 63) // 64
    x, wg, wu, wd = c.wide()
    fewer = ff.vjp(x[:rows], wg, wu, wd, *[v[:rows] for v in args[:3]], "silu")
    for n in (1, 2, 3):
        difference, of = off(outs[n], fewer[n])
        assert difference > 4 * limit[outs[n].dtype] * of, n
    narrow = ff.vjp(x, wg[:hidden], wu[:hidden], wd[:, :hidden], args[0][:, :hidden], args[1][:, :hidden], *args[2:])
    difference, of = off(outs[0], narrow[0])
    assert difference > 4 * limit[outs[0].dtype] * of


def test_many_calls_in_a_row():
    """Calls whose kernels take pairs of blocks and single ones by turns, each starting up while the one before ends, all
    of them with tensor memory: a thousand one after another give the bits of one alone."""
    import torch

    cases = [Case("f16", 5182, 1913, 69, "gelu"), Case("bf16", 300, 640, 520, gradient="f32"),
             Case("bf16", 40, 640, 520), Case("f16", 700, 24, 1000, gradient="f32")]
    want = []
    for c in cases:
        a, u, y, _ = c.forward()
        want.append((a, u, y, *c.vjp(a, u)[0]))
    torch.cuda.synchronize()
    p, L, stream = ff.pointer, abi.lib(), torch.cuda.current_stream().cuda_stream
    outs = [[torch.empty_like(v) for v in w] for w in want]
    for n in range(250):
        for c, o, w in zip(cases, outs, want):
            args = (ref(c.config), p(c.x), p(c.wg), p(c.wu), p(c.wd))
            assert L.geo_b200_feed_forward(*args, p(o[0]), p(o[1]), p(o[2]), p(c.space), c.space.numel(), stream) == 0
            assert L.geo_b200_feed_forward_vjp(*args, p(w[0]), p(w[1]), p(c.dy), *[p(v) for v in o[3:]], p(c.vjp_space),
                                               c.vjp_space.numel(), stream) == 0
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(v, e) for v, e in zip(o, w))


@pytest.mark.parametrize("gradient", ["f32", "f16"])
@pytest.mark.parametrize("rows,before", [(3, 0), (200, 0), (200, 1)])
def test_some_float16_cotangents(rows, before, gradient):
    """Each cotangent has the same bits alone as among all, whatever the powers of two are taken from."""
    import torch

    c = Case("f16", rows, 72, 136, gradient=None if gradient == "f16" else gradient, before=before)
    a, u, _, _ = c.forward()
    outs, _ = c.vjp(a, u)
    c.check_vjp(a, u, outs)
    for wanted in [(True, False, False, False), (False, True, False, False), (False, False, True, False),
                   (False, False, False, True), (True, False, True, True)]:
        again, _ = c.vjp(a, u, wanted=wanted)
        for on, one, other in zip(wanted, again, outs):
            assert torch.equal(one, other) if on else one.isnan().all()


@pytest.mark.parametrize("kind,limit", [("bf16", 2.0 ** -18), ("f16", 2.0 ** -19)])
def test_float32_cotangents_over_long_sums(kind, limit):
    """2-norms over 4096 columns and 8192 rows. Two terms leave at most 2^-18 of an inner value, 2^-18 / sqrt(3) of many
    (float16's: nothing that counts); the up to 32 instructions of a part of h_bar's and a cotangent's sums (float16: 16)
    cut some 2e-8 each; functions and the parts' own roundings leave 2^-21: below 2^-18, and 2^-19."""
    c = Case(kind, 8192, 4096, 256, gradient="f32")
    a, u, _, _ = c.forward()
    outs, _ = c.vjp(a, u)
    want = ff.vjp(*c.wide(), a.double(), u.double(), c.dy.double(), "silu")
    for n in (1, 2, 3):
        difference, of = off(outs[n], want[n])
        assert difference <= limit * of, n
