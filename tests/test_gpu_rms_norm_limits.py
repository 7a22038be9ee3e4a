"""The block norm's waits of clusters (geo/geo_b200.h section 5) on the GPU, made to give up."""
from __future__ import annotations

import ctypes

import pytest

import feed_forward_reference as ff
from geometricelementaryoperators_b200 import abi
from test_gpu_feed_forward import made

pytestmark = pytest.mark.gpu
ref, INVALID = ctypes.byref, 1


def stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


class Rows:
    """A block norm without gate and weights of packed float32 rows, its results, and the self-test's."""

    def __init__(self, rows, cols):
        import torch

        self.rows, self.cols = rows, cols
        self.x, self.residual, self.dy = (made(i, torch.float32, rows, cols) for i in range(3))
        self.config = abi.BlockNormConfig(type=abi.F32, parameter_type=abi.F32, gate=abi.GATE_NONE, rows=rows, cols=cols,
                                          epsilon=1e-5, residual_scale=0.75, block_scale=1.5)
        self.size = abi.lib().geo_b200_block_norm_vjp_workspace(ref(self.config))
        self.space = torch.empty(self.size, device="cuda", dtype=torch.uint8)
        self.clean = self.forward()
        self.clean_vjp = self.vjp()

    def new(self, *shape):
        import torch

        return torch.full(shape, 7.0, device="cuda")

    def outs(self):
        return [self.new(self.rows, self.cols), self.new(self.rows, self.cols), self.new(self.rows), self.new(self.rows)]

    def forward(self, round=None, polls=1 << 14):
        p, L, o = ff.pointer, abi.lib(), self.outs()
        if round is None:
            status = L.geo_b200_block_norm(ref(self.config), p(self.x), p(self.residual), None, None, None,
                                           *[p(v) for v in o], stream())
        else:
            status = L.geo_b200_block_norm_wait_selftest(ref(self.config), p(self.x), p(self.residual), None,
                                                         *[p(v) for v in o], None, None, None, 0, round, polls, stream())
        assert status == 0
        return o

    def vjp(self, round=None, polls=1 << 14):
        p, L = ff.pointer, abi.lib()
        z, _, x_rstd, z_rstd = self.clean
        o = self.outs()[:2] + [self.new(self.cols), self.new(self.cols)]
        if round is None:
            status = L.geo_b200_block_norm_vjp(ref(self.config), p(self.x), None, p(z), None, None, p(x_rstd), p(z_rstd),
                                               p(self.dy), None, p(o[0]), p(o[1]), None, p(o[2]), p(o[3]), p(self.space),
                                               self.size, stream())
        else:
            status = L.geo_b200_block_norm_wait_selftest(ref(self.config), p(self.x), p(z), p(self.dy), p(o[0]), p(o[1]),
                                                         p(x_rstd), p(z_rstd), p(o[2]), p(o[3]), p(self.space),
                                                         self.size, round, polls, stream())
        assert status == 0
        return o


@pytest.mark.parametrize("cols", [8192, 32768])
def test_block_norm_waits_give_up(cols):
    """Rows before the one that a block sends nothing for are right, it and those after it are NaN; the next call is
    right. A cluster's rows are as many apart as there are clusters; each takes two sums."""
    import torch

    r = Rows(700, cols)
    for round in (2, 3, 4):
        z, y, x_rstd, z_rstd = r.forward(round)
        torch.cuda.synchronize()
        first = int(y.isnan().any(1).int().argmax())
        step = first // (round // 2)
        assert 0 < first < r.rows and first % (round // 2) == 0
        for got, want in ((y, r.clean[1]), (z_rstd, r.clean[3])):
            assert torch.equal(got[:first], want[:first]) and got[first:].isnan().all()
        if round % 2:  # the row's first sum was whole, its second was not
            first += step
        for got, want in ((z, r.clean[0]), (x_rstd, r.clean[2])):
            assert torch.equal(got[:first], want[:first]) and got[first:].isnan().all()
    assert all(torch.equal(v, w) for v, w in zip(r.forward(1 << 20), r.clean))
    assert all(torch.equal(v, w) for v, w in zip(r.forward(), r.clean))


@pytest.mark.parametrize("cols", [8192, 32768])
def test_block_norm_vjp_waits_give_up(cols):
    import torch

    r = Rows(700, cols)
    for round in (1, 2):
        dresidual, dx, dpost, dpre = r.vjp(round)
        torch.cuda.synchronize()
        first = int(dx.isnan().any(1).int().argmax())
        assert 0 < first < r.rows and first % round == 0
        for got, want in ((dresidual, r.clean_vjp[0]), (dx, r.clean_vjp[1])):
            assert torch.equal(got[:first], want[:first]) and got[first:].isnan().all()
        assert dpost.isnan().all() and dpre.isnan().all()
    assert all(torch.equal(v, w) for v, w in zip(r.vjp(1 << 20), r.clean_vjp))
    assert all(torch.equal(v, w) for v, w in zip(r.vjp(), r.clean_vjp))


def test_block_norm_wait_selftest_refusals():
    p, L, r = ff.pointer, abi.lib(), Rows(4, 8192)
    o = [p(v) for v in r.outs()]

    def call(polls=1 << 14, z=p(r.residual), dy=None, **change):
        c = abi.BlockNormConfig(**{**{n: getattr(r.config, n) for n, _ in abi.BlockNormConfig._fields_}, **change})
        return L.geo_b200_block_norm_wait_selftest(ref(c), p(r.x), z, dy, *o, None, None, None, 0, 1 << 20, polls,
                                                   stream())

    assert call() == 0 and call(polls=1 << 22) == 0
    for bad in (dict(polls=0), dict(polls=(1 << 22) + 1), dict(z=None), dict(dy=p(r.dy)), dict(cols=4096),
                dict(cols=8188), dict(type=abi.F64, parameter_type=abi.F64), dict(gate=abi.GATE_SIGMOID),
                dict(x_stride=8192), dict(epsilon=-1.0)):
        assert call(**bad) == INVALID, bad
