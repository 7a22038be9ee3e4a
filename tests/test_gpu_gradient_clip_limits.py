"""Norm over a model's gradients and clipping (geo/geo_b200.h section 6) at its limits on the GPU."""
from __future__ import annotations

import pytest

from layer_reference import torch_type
from test_gpu_feed_forward import made
from test_gpu_gradient_clip import CLOSE, clip, norm_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [(1,), (2,), (64, 64, 65), (4096, 4097), (3_000_000, 17)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_squares_are_exact(kind, sizes):
    """No square of a type of up to 32 bits is rounded before it is summed in float64."""
    g = [made(i, torch_type(kind), n) for i, n in enumerate(sizes)]
    want = norm_of(g)
    assert abs(clip(g, 1.0, None)[0] - want) <= CLOSE * want


@pytest.mark.parametrize("outs", ["apart", "in place", None])
@pytest.mark.parametrize("sizes,others", [
    ((1e160,), ()), ((1e-170,), ()), ((1e300, 1e-300), ()), ((1e160, 1.0), ("f32", "bf16")), ((1e-170, 1e-150), ()),
    ((2.0 ** 480, 2.0 ** 482), ()), ((2.0 ** -480, 2.0 ** -482), ()), ((1e-200, 1e-30), ("f16",)), ((5e-324,), ()),
    ((2.0 ** -600,), ("f32",)), ((0.0, 1e-180, 0.0), ())])
def test_float64_beyond_its_squares(sizes, others, outs):
    """Float64 gradients whose squares leave float64's range, in whole pieces and in parts of some, alone and among
    others: the norm and the clipped values as for any."""
    import torch

    g = [made(i, torch.float64, 5000 + i).mul_(v) for i, v in enumerate(sizes)]
    g += [made(9 + i, torch_type(k), 300) for i, k in enumerate(others)]
    before = [v.clone() for v in g]
    back = 2.0 ** float(torch.stack([v.double().abs().max() for v in g]).max().log2().floor().clamp(min=-1000.0))
    want = norm_of([v.double() / back for v in g]) * back
    # A value as small as float64's least has no digits, and its quotient by 2^-1000 none of its own.
    norm, scale, clipped = clip(g, float(want) / 4, outs)
    assert want > 0 and abs(norm - want) <= CLOSE * want + 5e-324
    assert abs(scale - 0.25) <= 0.25 * (2 * CLOSE + (0.1 if want < 1e-310 else 0.0))
    for b, o in zip(before, clipped):
        if o is not None and b.dtype == torch.float64:
            assert torch.equal(o, b * scale)


def test_a_norm_beyond_float64():
    """Finite gradients whose norm is not: infinite, and scale NaN."""
    import torch

    g = [torch.full((100,), 1e308, device="cuda", dtype=torch.float64)]
    norm, scale, clipped = clip(g, 1.0)
    assert norm.isinf() and scale.isnan() and clipped[0].isnan().all()
    g[0][3] = float("nan")
    assert clip(g, 1.0)[0].isnan()


@pytest.mark.parametrize("outs", ["apart", "in place"])
@pytest.mark.parametrize("most", [1e-7, 1e-12, 1e-18])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_scales_below_float32(kind, most, outs):
    """Gradients of some 1e30 clipped to a small norm: scale has no digits, or is 0, in float32, and the clipped values
    are ordinary ones. The product is rounded to float32 and to the type."""
    import torch

    g = [made(1, torch_type(kind), 10007).mul_(1e30), made(2, torch_type(kind), 3).mul_(1e30)]
    before = [v.clone() for v in g]
    norm, scale, clipped = clip(g, most, outs)
    assert 0 < scale < 2.0 ** -126
    for b, o in zip(before, clipped):
        want = b.double() * scale
        t = torch.finfo(o.dtype).eps / 2 + 2.0 ** -24
        assert ((o.double() - want).abs() <= t * want.abs() + torch.finfo(torch.float32).smallest_normal * t).all()
    assert abs(norm_of(clipped) - most) <= most * (2.0 ** -7 if kind == "bf16" else 2.0 ** -22)
