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
