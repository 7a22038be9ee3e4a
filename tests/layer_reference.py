"""64-bit definitions of the layer operators (geo/geo_b200.h section 5) and the rounding bounds of the tests.

u(t) is half a step of type t relative to a value. A bound is u(type) |result| for the one final rounding plus a
number of roundings of the arithmetic type (float64 for float64, else float32) times what those roundings act on.
"""
from __future__ import annotations

import ctypes

import numpy as np

from geometricelementaryoperators_b200 import abi

TYPES = {"f64": abi.F64, "f32": abi.F32, "bf16": abi.BF16, "f16": abi.F16}


def torch_type(name):
    import torch

    return {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def half_step(dtype) -> float:
    import torch

    return torch.finfo(dtype).eps / 2


def least(dtype) -> float:
    """Half the smallest subnormal: the rounding of a result below the normal range."""
    import torch

    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps / 2


def wide_type(dtype):
    import torch

    return torch.float64 if dtype == torch.float64 else torch.float32


def u_wide(dtype) -> float:
    return half_step(wide_type(dtype))


def philox(block, offset, seed):
    """Philox4x32-10 of the counters (block, offset) under the key `seed`: an array [..., 4] of 32-bit words."""
    m, s = np.uint64(0xFFFFFFFF), np.uint64(32)
    b = np.asarray(block, dtype=np.uint64)
    c = [b & m, b >> s, np.full_like(b, offset & 0xFFFFFFFF), np.full_like(b, (offset >> 32) & 0xFFFFFFFF)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> s) ^ c[1] ^ np.uint64(k[0]), p1 & m, (p0 >> s) ^ c[3] ^ np.uint64(k[1]), p0 & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1)


def threshold(rate: float) -> int:
    return int(np.rint(rate * 65536.0))


def kept(rows, cols, dimension, rate, seed, offset, first_row=0):
    """Boolean [rows][cols]: the values that dropout keeps, rows first_row .. first_row + rows - 1."""
    e = np.arange(first_row * cols, (first_row + rows) * cols, dtype=np.uint64)
    unit = e >> np.uint64(dimension)
    first, last = int(unit[0]) >> 3, int(unit[-1]) >> 3
    words = philox(np.arange(first, last + 1, dtype=np.uint64), offset, seed)
    draws = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], -1).reshape(-1)
    at = (unit - np.uint64(first * 8)).astype(np.int64)
    return (draws[at] >= threshold(rate)).reshape(rows, cols)


def scale(rate: float) -> float:
    t = threshold(rate)
    return 65536.0 / (65536.0 - t) if t < 65536 else 0.0


def norm(x, weight, bias, eps):
    """Layer norm of a float64 tensor: y, mean, rstd."""
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1 / (d.square().mean(1) + eps).sqrt()
    y = d * rstd[:, None]
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return y, mean, rstd


#: Additions along the longest path of a row's sum: values a thread adds one after another, then the tree over
#: threads. 128 holds for rows of up to 16384 values (64 values for each of 256 threads, 5 steps in a warp, 8 warps).
PATH = 128


def norm_bound(x, weight, bias, rstd, y, dtype, path=PATH):
    """y, mean and rstd bounds. mean: `path` roundings of partial sums of at most cols mean|x|. rstd: half of the
    variance's `path` + 4 and its own 3. y = (x - mean) rstd weight + bias: those, and 4 of its own."""
    u = u_wide(dtype)
    average = x.abs().mean(1, keepdim=True)
    r = rstd[:, None]
    w = weight.abs() if weight is not None else 1.0
    hat = (x - x.mean(1, keepdim=True)).abs() * r * w
    b = bias.abs() if bias is not None else 0.0
    of_mean = path * u * average
    # The mean's error moves the variance by its square only.
    y_bound = half_step(dtype) * y.abs() + least(dtype) + of_mean * r * w + u * ((path / 2 + 9) * hat + 2 * b)
    y_bound = y_bound + hat * (of_mean * r).square()
    return y_bound, of_mean[:, 0], rstd * (u * (path / 2 + 6)) + rstd * (of_mean[:, 0] * rstd).square()


def norm_vjp(x, weight, mean, rstd, dy):
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy * weight if weight is not None else dy
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def norm_vjp_bound(x, weight, mean, rstd, dy, dx, dtype, path=PATH):
    """x_bar: `path` roundings of each of the two means (of |g| and |g xh|), 8 of its own terms. Column sums: a
    path of at most one rounding per row of a block plus the blocks, bounded by rows + 8 and by 700 (at most 512
    rows follow one another in a thread, then threads and blocks)."""
    u = u_wide(dtype)
    xh = (x - mean[:, None]).abs() * rstd[:, None]
    g = (dy * weight if weight is not None else dy).abs()
    along = (g * xh).mean(1, keepdim=True)
    dx_bound = half_step(dtype) * dx.abs() + least(dtype) + u * rstd[:, None] * (
        path * (g.mean(1, keepdim=True) + xh * along) + 8 * (g + xh * along))
    rows = min(x.shape[0] + 8, 700)
    return dx_bound, u * (rows + 4) * (dy.abs() * xh).sum(0), u * rows * dy.abs().sum(0)


def rotary_turns(rotary_dim, base=10000.0, scaling="none", factor=1.0, original=1.0, low=0.0, high=1.0):
    """Turns per position of each pair, in extended precision."""
    i = np.arange(rotary_dim // 2, dtype=np.longdouble)
    base, factor, d = np.longdouble(base), np.longdouble(factor), np.longdouble(rotary_dim)
    if scaling == "base" and rotary_dim > 2:
        base = base * factor ** (d / (d - 2))
    f = base ** (-2 * i / d)
    two_pi = 8 * np.arctan(np.longdouble(1))
    if scaling == "linear":
        f = f / factor
    if scaling == "banded":
        keep = np.clip((np.longdouble(original) * f / two_pi - np.longdouble(low)) / np.longdouble(high - low), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f / two_pi


def rotary(x, positions, turns, layout, amplitude, backward=False):
    """Rotates [batch][tokens][heads][head_dim] (float64 tensor); positions [batch][tokens] of Python integers."""
    import torch

    t = np.asarray(positions).astype(np.longdouble)[..., None] * turns
    t = (t - np.rint(t)) * (8 * np.arctan(np.longdouble(1)))
    to = lambda a: torch.tensor(a.astype(np.float64) * amplitude, device=x.device)[:, :, None]  # noqa: E731
    cos, sin = to(np.cos(t)), to(np.sin(t))
    if backward:
        sin = -sin
    r = 2 * len(turns)
    out = x.clone()
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if layout == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    u, v = a * cos - b * sin, a * sin + b * cos
    if layout == "half":
        out[..., :r // 2], out[..., r // 2:r] = u, v
    else:
        out[..., 0:r:2], out[..., 1:r:2] = u, v
    return out


def rotary_bound(x, y, turns, layout, amplitude, dtype, far):
    """Each result is a c - b s with |c|, |s| <= amplitude: 2 roundings each for sine and cosine (4 in float64, whose
    functions are within 2 steps), 1 for the amplitude, 2 for product and sum, 1 for the angle's conversion; and the
    angle's own error, 2 pi far turns 2^-62, and 2^-52 of float64 rounding."""
    r = 2 * len(turns)
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if layout == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    size = (a.abs() + b.abs()) * abs(amplitude)
    import torch

    angle = 2 * np.pi * (float(far) * turns.astype(np.float64) * 2.0 ** -62 + 2.0 ** -52)
    each = size * (10 * u_wide(dtype) + torch.tensor(angle, device=x.device))
    bound = torch.zeros_like(x)
    if layout == "half":
        bound[..., :r // 2], bound[..., r // 2:r] = each, each
    else:
        bound[..., 0:r:2], bound[..., 1:r:2] = each, each
    bound[..., :r] += half_step(dtype) * y[..., :r].abs() + least(dtype)
    return bound


def pointer(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def assert_within(got, want, bound, what=""):
    import torch

    got = got.double()
    bad = ~((got - want).abs() <= bound)
    if bad.any():
        at = tuple(int(v) for v in torch.nonzero(bad)[0])
        worst = ((got - want).abs() / (bound + 1e-300)).max()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {at}: "
                             f"{float(got[at])} for {float(want[at])}, bound {float((bound + 0 * want)[at])}, "
                             f"worst {float(worst):.3g} of its bound")
