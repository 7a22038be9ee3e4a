"""Gated feed-forward block (geo/geo_b200.h section 5) at its limits on the GPU: waits that give up anywhere."""
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
