"""Norm over a model's gradients and clipping (geo/geo_b200.h section 6) on the GPU."""
from __future__ import annotations

import ctypes

import pytest

from geometricelementaryoperators_b200 import abi
from layer_reference import TYPES, torch_type
from test_gpu_feed_forward import made

pytestmark = pytest.mark.gpu

#: Float64 sums of non-negative terms: one rounding for each of at most 2^12 additions along a path, and the root's.
#: A float32 value's square is rounded to float32, 2^-24 of itself: no more than that of a sum of non-negative terms, and
#: half of it, 2^-25, of the sum's root.
CLOSE = 2.0 ** -40


def close_of(gradients):
    import torch

    return CLOSE + (2.0 ** -25 if any(g.dtype == torch.float32 and g.numel() for g in gradients) else 0.0)


def clip(gradients, max_norm, outs="apart", space=None, stream=None):
    """Calls the library; returns norm, scale and the clipped tensors."""
    import torch

    kinds = {torch_type(k): v for k, v in TYPES.items()}
    if outs == "apart":
        outs = [torch.full_like(g, float("nan")) for g in gradients]
    elif outs == "in place":
        outs = gradients
    elif outs is None:
        outs = [None] * len(gradients)
    table = (abi.Gradient * len(gradients))(*[
        abi.Gradient(type=kinds[g.dtype], count=g.numel(), gradient=g.data_ptr() or None,
                     clipped=None if o is None else (o.data_ptr() or None)) for g, o in zip(gradients, outs)])
    L = abi.lib()
    size = L.geo_b200_gradient_clip_workspace(table, len(gradients))
    assert size > 0
    if space is None:
        space = torch.empty(size, device="cuda", dtype=torch.uint8)
    found = torch.full((2,), float("nan"), device="cuda", dtype=torch.float64)
    status = L.geo_b200_gradient_clip(table, len(gradients), max_norm, found.data_ptr(), found.data_ptr() + 8,
                                      space.data_ptr(), size,
                                      stream if stream is not None else torch.cuda.current_stream().cuda_stream)
    assert status == 0
    return found[0], found[1], outs


def norm_of(gradients):
    import torch

    return torch.sqrt(sum((g.double().square().sum() for g in gradients), torch.zeros((), device="cuda").double()))


def check(gradients, max_norm, norm, scale, outs, before=None):
    import torch

    want, close = norm_of(before or gradients), close_of(before or gradients)
    assert abs(norm - want) <= close * want
    assert abs(scale - min(1.0, max_norm / float(want)) if want > 0 else scale - 1.0) <= 2 * close
    for g, o in zip(before or gradients, outs):
        if o is None:
            continue
        wide = torch.float64 if g.dtype == torch.float64 else torch.float32
        assert torch.equal(o, (g.to(wide) * scale.to(wide)).to(g.dtype))


LISTS = {
    "one value": [("f32", 1)],
    "each type": [("f64", 1000), ("f32", 4099), ("bf16", 8192), ("f16", 40001)],
    "some empty": [("bf16", 0), ("f32", 17), ("f16", 0), ("f64", 3), ("bf16", 0)],
    "many small": [(k, 1 + 37 * i % 200) for i in range(400) for k in ("f64", "bf16")][:700],
    "several launches": [("bf16", 1 + i % 5) for i in range(2500)] + [("f32", 100000)],
    "pieces": [("bf16", 8191), ("bf16", 8192), ("bf16", 8193), ("f32", 4095), ("f32", 4096), ("f32", 4097),
               ("f64", 2048), ("f64", 2049), ("f16", 16385)],
    "large": [("bf16", 20_000_003), ("f32", 9_999_999), ("f16", 123)],
}


@pytest.mark.parametrize("outs", ["apart", "in place", None])
@pytest.mark.parametrize("name", list(LISTS))
def test_lists(name, outs):
    gradients = [made(i, torch_type(k), n) for i, (k, n) in enumerate(LISTS[name])]
    before = [g.clone() for g in gradients]
    norm = float(norm_of(gradients))
    for most in (0.3 * norm, 2 * norm):
        for g, b in zip(gradients, before):
            g.copy_(b)
        check(gradients, most, *clip(gradients, most, outs), before=before)


@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("offset", [1, 3])
def test_parts_of_a_buffer(kind, offset):
    """Gradients that start off 16 bytes, side by side in one buffer; what lies between them stays."""
    import torch

    sizes, gap = [5, 1000, 20000, 7, 33333], 2
    buffer = made(1, torch_type(kind), offset + sum(sizes) + gap * len(sizes))
    out, parts, clipped, at = torch.full_like(buffer, 3.0), [], [], offset
    kept = torch.ones(buffer.numel(), dtype=torch.bool, device="cuda")
    for n in sizes:
        parts.append(buffer[at:at + n])
        clipped.append(out[at:at + n])
        kept[at:at + n] = False
        at += n + gap
    check(parts, 1.0, *clip(parts, 1.0, clipped))
    assert (out[kept] == 3.0).all()


def test_ranges_of_the_types():
    """Squares beyond float32's range on both sides, in a sum that is float64."""
    import torch

    for value in (1e30, 1e-30):
        g = [torch.full((5000,), value, device="cuda", dtype=torch.bfloat16), torch.full((77,), value, device="cuda")]
        norm, scale, outs = clip(g, value)
        check(g, value, norm, scale, outs)
        assert norm > 0 and scale < 1


def test_zero_infinite_and_nan():
    import torch

    zero = [torch.zeros(100, device="cuda"), torch.zeros(3, device="cuda", dtype=torch.float16)]
    norm, scale, outs = clip(zero, 1.0)
    assert norm == 0 and scale == 1 and all((o == 0).all() for o in outs)
    some = [made(1, torch.float32, 1000)]
    norm, scale, outs = clip(some, float("inf"))
    assert scale == 1 and torch.equal(outs[0], some[0])
    for bad in (float("inf"), float("nan")):
        some[0][17] = bad
        norm, scale, outs = clip(some, 1.0)
        assert not norm.isfinite() and scale.isnan() and outs[0].isnan().all()


def test_same_bits_captured_and_on_streams():
    import torch

    lists = [[made(10 * i + j, t, n) for j, (t, n) in enumerate(((torch.bfloat16, 3_000_000), (torch.float32, 12345)))]
             for i in range(2)]
    first = [clip(g, 1.0) for g in lists]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = [clip(g, 1.0, stream=s.cuda_stream) for g, s in zip(lists, streams)]
        torch.cuda.synchronize()
        for (n, s, o), (wn, ws, wo) in zip(got, first):
            assert n == wn and s == ws and all(torch.equal(a, b) for a, b in zip(o, wo))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, scale, outs = clip(lists[0], 1.0)
    for g, b in zip(lists[0], lists[1]):
        g.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    assert norm == first[1][0] and scale == first[1][1] and all(torch.equal(a, b) for a, b in zip(outs, first[1][2]))


def test_overlaps():
    """What is written overlaps nothing else; what is only read may be listed twice and counts twice."""
    import torch

    L = abi.lib()
    g = made(1, torch.float32, 1000)
    out = torch.empty(1000, device="cuda")
    space = torch.empty(1 << 16, device="cuda", dtype=torch.uint8)

    def call(*entries):
        t = (abi.Gradient * len(entries))(*[abi.Gradient(type=abi.F32, count=n, gradient=a, clipped=c)
                                            for n, a, c in entries])
        return L.geo_b200_gradient_clip(t, len(entries), 1.0, None, None, space.data_ptr(), space.numel(),
                                        torch.cuda.current_stream().cuda_stream)

    a, o = g.data_ptr(), out.data_ptr()
    assert call((500, a, a), (500, a + 2000, a + 2000)) == 0
    assert call((1000, a, o)) == 0
    assert call((1000, a, a), (1000, a, a)) == 1
    assert call((1000, a, o), (500, a, o + 2000)) == 1
    assert call((600, a, a), (500, a + 2000, None)) == 1
    assert call((500, a, a + 4)) == 1
    assert call((500, a, o), (500, o, None)) == 1
    host = torch.empty(1000)
    assert call((1000, host.data_ptr(), None)) == 1 and call((1000, a, host.data_ptr())) == 1
    assert call((1000, a + 2, None)) == 1
    torch.cuda.synchronize()
    norm, _, _ = clip([g, g], 1.0, None)
    assert abs(norm - norm_of([g, g])) <= close_of([g]) * norm


def test_a_layer_is_trained():
    """The operators together, as one half of a layer uses them: norm, feed-forward block, block norm, their VJPs, and
    the clipping of all gradients. The gradients against central differences of the loss in float64."""
    import torch

    import feed_forward_reference as ff

    rows, cols, hidden, eps = 40, 64, 96, 1e-5
    L, ref, p = abi.lib(), ctypes.byref, ff.pointer
    f64 = torch.float64
    shapes = {"x": (rows, cols), "gate": (rows, cols), "wg": (hidden, cols), "wu": (hidden, cols), "wd": (cols, hidden),
              "first": (cols,), "post": (cols,), "pre": (cols,)}
    t = {n: made(i, f64, *s, scale=1.0 if len(s) == 2 and s[0] == rows else 0.1)
         for i, (n, s) in enumerate(shapes.items())}
    dy, dz = made(20, f64, rows, cols), made(21, f64, rows, cols)

    def loss(t):
        h, _ = ff.rms(t["x"], t["first"], eps)
        y = ff.forward(h, t["wg"], t["wu"], t["wd"], "silu")[2]
        z, out, _, _ = ff.block(y, t["x"], t["gate"], "sigmoid", t["post"], t["pre"], 1.0, 0.5, eps)
        return (out * dy).sum() + (z * dz).sum()

    new = lambda *s: torch.empty(*s, device="cuda", dtype=f64)  # noqa: E731
    norm = abi.LayerNormConfig(type=abi.F64, parameter_type=abi.F64, rows=rows, cols=cols, epsilon=eps)
    feed = abi.FeedForwardConfig(type=abi.F64, gradient_type=abi.F64, activation=abi.ACTIVATION_SILU, rows=rows,
                                 cols=cols, hidden=hidden)
    join = abi.BlockNormConfig(type=abi.F64, parameter_type=abi.F64, gate=abi.GATE_SIGMOID, rows=rows, cols=cols,
                               epsilon=eps, residual_scale=1.0, block_scale=0.5)
    sizes = [L.geo_b200_rms_norm_vjp_workspace(ref(norm)), L.geo_b200_feed_forward_workspace(ref(feed)),
             L.geo_b200_feed_forward_vjp_workspace(ref(feed)), L.geo_b200_block_norm_vjp_workspace(ref(join))]
    space = torch.empty(max(sizes), device="cuda", dtype=torch.uint8)
    s = torch.cuda.current_stream().cuda_stream
    h, rstd, a, u, y, z, out, y_rstd, z_rstd = (new(rows, cols), new(rows), new(rows, hidden), new(rows, hidden),
                                                new(rows, cols), new(rows, cols), new(rows, cols), new(rows), new(rows))
    grads = {n: new(*v) for n, v in shapes.items()}
    dblock, dfeed, dres = new(rows, cols), new(rows, cols), new(rows, cols)
    status = [
        L.geo_b200_rms_norm(ref(norm), p(t["x"]), p(t["first"]), p(h), p(rstd), s),
        L.geo_b200_feed_forward(ref(feed), p(h), p(t["wg"]), p(t["wu"]), p(t["wd"]), p(a), p(u), p(y), p(space), sizes[1], s),
        L.geo_b200_block_norm(ref(join), p(y), p(t["x"]), p(t["gate"]), p(t["post"]), p(t["pre"]), p(z), p(out),
                              p(y_rstd), p(z_rstd), s),
        L.geo_b200_block_norm_vjp(ref(join), p(y), p(t["gate"]), p(z), p(t["post"]), p(t["pre"]), p(y_rstd), p(z_rstd),
                                  p(dy), p(dz), p(dres), p(dblock), p(grads["gate"]), p(grads["post"]), p(grads["pre"]),
                                  p(space), sizes[3], s),
        L.geo_b200_feed_forward_vjp(ref(feed), p(h), p(t["wg"]), p(t["wu"]), p(t["wd"]), p(a), p(u), p(dblock), p(dfeed),
                                    p(grads["wg"]), p(grads["wu"]), p(grads["wd"]), p(space), sizes[2], s),
        L.geo_b200_rms_norm_vjp(ref(norm), p(t["x"]), p(t["first"]), p(rstd), p(dfeed), p(grads["x"]),
                                p(grads["first"]), p(space), sizes[0], s)]
    assert status == [0] * 6
    grads["x"] += dres
    for i, n in enumerate(shapes):
        d = made(40 + i, f64, *shapes[n])
        at = lambda e: loss({**t, n: t[n] + e * d})  # noqa: E731
        slope = (at(1e-5) - at(-1e-5)) / 2e-5
        # Third derivatives times 1e-10, rounding of the loss (1e-13 of some hundreds) over 1e-5.
        assert abs(slope - (grads[n] * d).sum()) <= 1e-6 * (grads[n] * d).abs().sum(), n
    held = [grads[n].clone() for n in shapes]
    found, scale, clipped = clip([grads[n] for n in shapes], 0.1, "in place")
    assert abs(found - norm_of(held)) <= CLOSE * found and abs(norm_of(clipped) - 0.1) <= 1e-12
