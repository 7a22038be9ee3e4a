"""64-bit definitions of the feed-forward block, RMS norm and the block norm (geo/geo_b200.h section 5), and the
rounding bounds of the tests. half_step and least are layer_reference's; u is half a step of the arithmetic type.

Sums of K products are bounded by 2 K u of the sum of their sizes: one rounding for each product and addition, and
tensor cores may cut where others round.
"""
from __future__ import annotations

import ctypes
import math

from geometricelementaryoperators_b200 import abi
from layer_reference import half_step, least, u_wide

ACTIVATIONS = {"silu": abi.ACTIVATION_SILU, "gelu": abi.ACTIVATION_GELU, "sigmoid": abi.ACTIVATION_SIGMOID,
               "relu": abi.ACTIVATION_RELU}
GATES = {"none": abi.GATE_NONE, "linear": abi.GATE_LINEAR, "sigmoid": abi.GATE_SIGMOID, "tanh": abi.GATE_TANH}


def activation(a, kind):
    """act(a) and act'(a)."""
    import torch

    if kind == "relu":
        return a.clamp(min=0), (a > 0).double()
    if kind == "gelu":
        phi = 0.5 * torch.erfc(-a / math.sqrt(2))
        return a * phi, phi + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    s, rest = torch.sigmoid(a), torch.sigmoid(-a)
    return (s, s * rest) if kind == "sigmoid" else (a * s, s * (1 + a * rest))


def function_error(a, u):
    """Relative error of act and act' terms: their argument's rounding grows with |a| in e^-a and a^2 in Phi and
    e^(-a^2/2); 16 roundings for the functions and what surrounds them (float32's fast exponential and division are
    within 2^-22 each)."""
    return u * (16 + 4 * a.abs() + 2 * a * a)


def forward(x, wg, wu, wd, kind):
    a, u = x @ wg.T, x @ wu.T
    f, _ = activation(a, kind)
    return a, u, (f * u) @ wd.T


def forward_bound(x, wg, wu, wd, kind, dtype):
    """Of gate, up and y. |act'| <= 1.2 for all four, so an argument off by d gives a value off by 1.2 d."""
    e, t, small = u_wide(dtype), half_step(dtype), least(dtype)
    a, u, y = forward(x, wg, wu, wd, kind)
    f, _ = activation(a, kind)
    da, du = 2 * x.shape[1] * e * (x.abs() @ wg.abs().T), 2 * x.shape[1] * e * (x.abs() @ wu.abs().T)
    h = (f * u).abs()
    dh = 1.2 * da * (u.abs() + du) + f.abs() * du + function_error(a, e) * h + t * h + small
    dy = dh @ wd.abs().T + 2 * wd.shape[1] * e * ((h + dh) @ wd.abs().T)
    return da + t * a.abs() + small, du + t * u.abs() + small, dy + t * (y.abs() + dy) + small


def vjp(x, wg, wu, wd, a, u, dy, kind):
    f, slope = activation(a, kind)
    dh = dy @ wd
    da, du = dh * u * slope, dh * f
    return da @ wg + du @ wu, da.T @ x, du.T @ x, dy.T @ (f * u)


def vjp_bound(x, wg, wu, wd, a, u, dy, kind, dtype, gradient_dtype):
    """Of x_bar and the three weights' cotangents. On their way to a float32 cotangent the inner values are two of
    their type: what is left off is half a step of half a step, and half of the type's least."""
    e, t, small = u_wide(dtype), half_step(dtype), least(dtype)
    rows, cols, hidden = x.shape[0], x.shape[1], wg.shape[0]
    f, slope = activation(a, kind)
    dh = dy @ wd
    da, du, h = dh * u * slope, dh * f, f * u
    off = 2 * cols * e * (dy.abs() @ wd.abs())
    fe = function_error(a, e)
    at = (u * slope).abs() * off + 2 * fe * (dh * u).abs() + 4 * e * da.abs()
    ut = f.abs() * off + (fe + 4 * e) * du.abs()
    ht = (fe + 4 * e) * h.abs()
    rounded = lambda d, v: d + t * (v.abs() + d) + small  # noqa: E731
    twice = lambda d, v: d + t * t * (v.abs() + d) + small  # noqa: E731
    ra, ru = rounded(at, da), rounded(ut, du)
    dx = da @ wg + du @ wu
    bound_x = ra @ wg.abs() + ru @ wu.abs() + 4 * hidden * e * ((da.abs() + ra) @ wg.abs() + (du.abs() + ru) @ wu.abs())
    inner = twice if gradient_dtype != dtype else rounded
    g = half_step(gradient_dtype)

    def weight(d, v, other):
        d = inner(d, v)
        return d.T @ other.abs() + 4 * rows * e * ((v.abs() + d).T @ other.abs())

    outs = [(da.T @ x, weight(at, da, x)), (du.T @ x, weight(ut, du, x)), (dy.T @ h, weight(ht, h, dy).T)]
    return (bound_x + t * (dx.abs() + bound_x) + small,
            *[b + g * (w.abs() + b) + least(gradient_dtype) for w, b in outs])


def gate_value(g, kind):
    import torch

    if kind == "linear":
        return g, torch.ones_like(g)
    if kind == "tanh":
        return torch.tanh(g), 1 / torch.cosh(g).square()
    return torch.sigmoid(g), torch.sigmoid(g) * torch.sigmoid(-g)


#: Additions along the longest path of a row's sum (layer_reference.PATH) and a column's.
PATH = 128


def rms(x, w, eps):
    rstd = 1 / (x.square().mean(1) + eps).sqrt()
    y = x * rstd[:, None]
    return (y if w is None else y * w), rstd


def rms_bound(y, rstd, dtype, path=PATH):
    u = u_wide(dtype)
    return half_step(dtype) * y.abs() + least(dtype) + u * (path / 2 + 8) * y.abs(), u * (path / 2 + 6) * rstd


def rms_vjp(x, w, rstd, dy):
    xh = x * rstd[:, None]
    g = dy if w is None else dy * w
    return rstd[:, None] * (g - xh * (g * xh).mean(1, keepdim=True)), (dy * xh).sum(0)


def column_path(rows):
    """Roundings of a column's sum: at most 512 rows follow one another in a thread, then threads and blocks."""
    return min(rows + 8, 700)


def rms_vjp_bound(x, w, rstd, dy, dx, dtype, path=PATH):
    u = u_wide(dtype)
    xh = (x * rstd[:, None]).abs()
    g = (dy if w is None else dy * w).abs()
    along = (g * xh).mean(1, keepdim=True)
    bound = half_step(dtype) * dx.abs() + least(dtype) + u * rstd[:, None] * ((path + 8) * xh * along + 8 * g)
    return bound, u * (column_path(x.shape[0]) + 4) * (dy.abs() * xh).sum(0)


def one(w):
    return 1.0 if w is None else w


def block(x, residual, gate, kind, post, pre, alpha, beta, eps):
    n, x_rstd = rms(x, post, eps)
    if gate is not None:
        n = n * gate_value(gate, kind)[0]
    z = alpha * residual + beta * n
    y, z_rstd = rms(z, pre, eps)
    return z, y, x_rstd, z_rstd


def block_bound(x, residual, gate, kind, post, pre, alpha, beta, eps, dtype, path=PATH):
    u, t, small = u_wide(dtype), half_step(dtype), least(dtype)
    z, y, x_rstd, z_rstd = block(x, residual, gate, kind, post, pre, alpha, beta, eps)
    n = (z - alpha * residual).abs()
    extra = 0 if gate is None else 16 + 4 * gate.abs()
    of_z = u * (2 * (alpha * residual).abs() + (path / 2 + 16 + extra) * n)
    # The statistic of z moves by the relative error of its squares' mean.
    moved = (z.abs() * of_z + of_z.square()).mean(1, keepdim=True) * z_rstd[:, None].square()
    of_y = of_z * z_rstd[:, None] * abs_of(pre) + y.abs() * (u * (path / 2 + 10) + moved)
    return (of_z + t * (z.abs() + of_z) + small, of_y + t * (y.abs() + of_y) + small,
            x_rstd * u * (path / 2 + 6), z_rstd * (u * (path / 2 + 6) + moved[:, 0]))


def abs_of(w):
    return 1.0 if w is None else w.abs()


def block_vjp(x, gate, kind, z, post, pre, x_rstd, z_rstd, dy, dz, alpha, beta):
    import torch

    dzs, dpre = rms_vjp(z, pre, z_rstd, dy)
    if dz is not None:
        dzs = dzs + dz
    f, slope = (torch.ones_like(x), None) if gate is None else gate_value(gate, kind)
    dx, dpost = rms_vjp(x, post, x_rstd, beta * f * dzs)
    dgate = None if gate is None else beta * dzs * x * x_rstd[:, None] * one(post) * slope
    return alpha * dzs, dx, dgate, dpost, dpre


def block_vjp_bound(x, gate, kind, z, post, pre, x_rstd, z_rstd, dy, dz, alpha, beta, dtype, path=PATH):
    """In sizes of terms: dz's own, d = rz (|g| + |zh| mean |g zh|) + |z_bar|, is off by path + 12 roundings of it, and
    the second mean by three sums' path and the products' few."""
    import torch

    u, t, small = u_wide(dtype), half_step(dtype), least(dtype)
    outs = block_vjp(x, gate, kind, z, post, pre, x_rstd, z_rstd, dy, dz, alpha, beta)
    zh, xh = (z * z_rstd[:, None]).abs(), (x * x_rstd[:, None]).abs()
    g = (dy * one(pre)).abs()
    d = z_rstd[:, None] * (g + zh * (g * zh).mean(1, keepdim=True)) + (0 if dz is None else dz.abs())
    off = u * (path + 12) * d
    f, slope, extra = torch.ones_like(x), torch.ones_like(x), torch.zeros_like(x)
    if gate is not None:
        f, slope = (v.abs() for v in gate_value(gate, kind))
        extra = 16 + 8 * gate.abs()
    beta, alpha, p = abs(beta), abs(alpha), abs_of(post)
    dn_off = beta * f * (off + u * (8 + extra) * d)
    along = (beta * f * p * xh * d).mean(1, keepdim=True)
    along_off = u * (3 * path + 24) * along + (beta * f * p * xh * u * extra * d).mean(1, keepdim=True)
    dx_off = x_rstd[:, None] * (p * dn_off + xh * along_off + 8 * u * (beta * f * p * d + xh * along))
    dg_off = beta * slope * p * xh * (off + u * (12 + extra) * d)
    rows = column_path(x.shape[0])
    dpost_off = (dn_off * xh).sum(0) + u * (rows + 4) * (beta * f * d * xh).sum(0)
    dpre_off = u * (rows + 4) * (dy.abs() * zh).sum(0)
    final = lambda v, b: b + t * (v.abs() + b) + small  # noqa: E731
    return (final(outs[0], alpha * off + 2 * u * alpha * d), final(outs[1], dx_off),
            None if gate is None else final(outs[2], dg_off), dpost_off, dpre_off)


def pointer(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None
