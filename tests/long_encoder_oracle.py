"""Plain 64-bit forms of the gated product, of products of 8-bit whole numbers and of windowed
attention, with bounds on what a kernel may be off that rounds where it has to (as in encoder_oracle,
whose units these are in).
"""

from __future__ import annotations

import math

import torch

import encoder_oracle as o


# ---- gated product ------------------------------------------------------------------


def activate(z, act):
    if act == "silu":
        return z * torch.special.expit(z)
    return torch.special.expit(z) if act == "sigmoid" else o.activate(z, act)


def slope(z, act):
    if act == "silu":
        s, rest = torch.special.expit(z), torch.special.expit(-z)
        return s * (1 + z * rest)
    return torch.special.expit(z) * torch.special.expit(-z) if act == "sigmoid" else o.slope(z, act)


def gated(x, wg, wu, bg, bu, act):
    """(y, pre)."""
    g, u = (x @ w.T + (0 if b is None else b) for w, b in ((wg, bg), (wu, bu)))
    return activate(g, act) * u, torch.cat([g, u], -1)


def gated_bounds(x, wg, wu, bg, bu, act, dtype):
    """Both sums' fp32 roundings (any order of k terms), an activation of slope at most 1.13 that is good to 1e-6,
    the product's and the result's rounding."""
    y, pre = gated(x, wg, wu, bg, bu, act)
    g, u = pre.chunk(2, -1)
    slip_g, slip_u = (o.F32 * (8 + math.sqrt(x.shape[-1])) * (x.abs() @ w.abs().T + (0 if b is None else b.abs()))
                      for w, b in ((wg, bg), (wu, bu)))
    h = activate(g, act).abs()
    off = 1.13 * slip_g + 1e-6 * (1 + h)
    return (o.U[dtype] * y.abs() + o.TINY[dtype] + off * (u.abs() + slip_u) + h * slip_u + 2 * o.F32 * y.abs(),
            o.U[dtype] * pre.abs() + o.TINY[dtype] + torch.cat([slip_g, slip_u], -1))


def _flat(t):
    return t.reshape(-1, t.shape[-1])


def gated_grads(dy, x, wg, wu, pre, act):
    """(dx, dgate, dup, dgate_bias, dup_bias)."""
    g, u = pre.chunk(2, -1)
    dg, du = dy * u * slope(g, act), dy * activate(g, act)
    return dg @ wg + du @ wu, _flat(dg).T @ _flat(x), _flat(du).T @ _flat(x), _flat(dg).sum(0), _flat(du).sum(0)


def gated_grad_bounds(dy, x, wg, wu, pre, act, dtype):
    """dg and du are rounded before the products, and come of values and slopes good to 1e-6 and 2e-6."""
    g, u = pre.chunk(2, -1)
    h = activate(g, act)
    dg, du = dy * u * slope(g, act), dy * h
    unit, tiny = o.U[dtype], o.TINY[dtype]
    eps_g = 2e-6 * (dy * u).abs() + 2 * o.F32 * dg.abs()
    eps_u = 1e-6 * dy.abs() * (1 + h.abs()) + o.F32 * du.abs()
    off_g, off_u = eps_g + unit * dg.abs() + tiny, eps_u + unit * du.abs() + tiny
    chain_x, chain_w = o.F32 * (8 + math.sqrt(2 * wg.shape[0])), o.F32 * (8 + math.sqrt(_flat(x).shape[0]))
    dx, dwg, dwu, dbg, dbu = gated_grads(dy, x, wg, wu, pre, act)
    xa = _flat(x).abs()

    def weight(d, off, want):
        return unit * want.abs() + tiny + (_flat(off).T + chain_w * _flat(d).abs().T) @ xa

    def bias(d, eps, want):
        return unit * want.abs() + tiny + _flat(eps).sum(0) + chain_w * _flat(d).abs().sum(0)

    return (unit * dx.abs() + tiny + (off_g + chain_x * dg.abs()) @ wg.abs() + (off_u + chain_x * du.abs()) @ wu.abs(),
            weight(dg, off_g, dwg), weight(du, off_u, dwu), bias(dg, eps_g, dbg), bias(du, eps_u, dbu))


# ---- 8-bit whole numbers --------------------------------------------------------------


def quantize(x):
    """(whole numbers, units in 64 bits) of the rows: 127 x / top to the nearest, ties to the even one."""
    top = x.abs().amax(-1, keepdim=True)
    odd = ~torch.isfinite(x).all(-1, keepdim=True)
    safe = torch.where(odd | (top == 0), torch.ones_like(top), top)
    values = torch.round(torch.where(odd, torch.zeros_like(x), x) * 127 / safe)
    return values, torch.where(odd, torch.full_like(top, math.nan), top / 127)[..., 0]


def linear_int8(x, values, scales, b, act, res):
    q, unit = quantize(x)
    z = (q @ values.T) * unit[..., None] * scales
    if b is not None:
        z = z + b
    y = o.activate(z, act)
    return (y if res is None else y + res), z


def linear_int8_bounds(x, values, scales, b, act, res, dtype):
    """Whole sums are exact; the conversion, the scale's rounding, two products, the bias: fp32 roundings of z's terms."""
    y, z = linear_int8(x, values, scales, b, act, res)
    bias = torch.zeros(()).double() if b is None else b
    slip = 6 * o.F32 * ((z - bias).abs() + bias.abs())
    return (o.U[dtype] * y.abs() + o.TINY[dtype] + 1.13 * slip + 1e-6 * (1 + o.activate(z, act).abs() if act else 0) + 2 * o.F32 * y.abs())
