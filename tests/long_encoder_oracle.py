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


# ---- attention with a window ------------------------------------------------------------


def window_seen(b, lq, lk, before, after, sinks, causal=False, key_lengths=None, query_lengths=None, query_start=None):
    """(positions key - row [b, lq, lk], which pairs are seen)."""
    start = torch.full((b,), lk - lq) if query_start is None else query_start.long().cpu()
    j = torch.arange(lk)
    rel = j[None, None, :] - torch.arange(lq)[None, :, None] - start[:, None, None]
    seen = ((rel >= -before) & (rel <= after)) | (j < sinks)
    if causal:
        seen = seen & (rel <= 0)
    if key_lengths is not None:
        seen = seen & (j[None, :] < key_lengths.long().cpu()[:, None])[:, None, :]
    if query_lengths is not None:
        seen = seen & (torch.arange(lq)[None, :] < query_lengths.long().cpu()[:, None])[:, :, None]
    return rel, seen


def window_attention(q, k, v, do, scale, dtype, before, after, sinks, table=None, max_distance=128, causal=False, own_delta=False,
                     **masks):
    """{"out", "lse", "dq", "dk", "dv", "dtable"}: (value, bound) of each, by the definition and its formulas.

    Bounds as encoder_oracle's: delta is off by the rounding of ``out``, or (``own_delta``) by its own fp32 sums only."""
    (b, lq, h, _), lk, hk = q.shape, k.shape[1], k.shape[2]
    rel, seen = window_seen(b, lq, lk, before, after, sinks, causal, **masks)
    keys, rows = seen.any(1)[:, :, None, None], seen.any(2)[:, :, None, None]
    zero = torch.zeros((), dtype=torch.float64)
    k, v = (torch.where(keys, t, zero).repeat_interleave(h // hk, 2).transpose(1, 2) for t in (k, v))
    q, g = (torch.where(rows, t, zero).transpose(1, 2) for t in (q, do))
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    found = None
    if table is not None:
        found = o.bucket(rel, table.shape[0], causal, max_distance)
        s = s + table[found].permute(0, 3, 1, 2)
    s = s.masked_fill(~seen[:, None], -math.inf)
    lse = torch.logsumexp(s, 3)
    none = torch.isinf(lse)
    p = torch.exp(s - torch.where(none, zero, lse)[..., None])
    u, tiny = o.U[dtype], o.TINY[dtype]
    out = torch.matmul(p, v)
    bound = u * out.abs() + tiny + (u + o.SCORE) * torch.matmul(p, v.abs()) + tiny * v.abs().sum(2, keepdim=True)
    res = {"out": (out.transpose(1, 2), bound.transpose(1, 2)),
           "lse": (lse, 2.0**-17 + 2.0**-20 * torch.where(none, zero, lse).abs())}
    dp = torch.matmul(g, v.transpose(2, 3).contiguous())
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    size = torch.matmul(g.abs(), v.abs().transpose(2, 3).contiguous())
    if own_delta:
        slip = 2.0**-20 * (p * size).sum(3, keepdim=True)
    else:
        slip = u * (g * out).abs().sum(3, keepdim=True) + tiny * g.abs().sum(3, keepdim=True)
    off = o.SCORE * ds.abs() + p * (slip + 2.0**-20 * size)  # of ds, before it is rounded
    inner, round_p = off + u * ds.abs() + tiny, o.SCORE * p + u * p + tiny

    def share(t):
        return t.transpose(1, 2).reshape(b, lk, hk, h // hk, -1).sum(3)

    def t23(t):
        return t.transpose(2, 3).contiguous()

    for name, value, more in (("dq", (torch.matmul(ds, k) * scale).transpose(1, 2), scale * torch.matmul(inner, k.abs()).transpose(1, 2)),
                              ("dk", share(torch.matmul(t23(ds), q)) * scale, scale * share(torch.matmul(t23(inner), q.abs()))),
                              ("dv", share(torch.matmul(t23(p), g)), share(torch.matmul(t23(round_p), g.abs())))):
        res[name] = value, u * value.abs() + tiny + more
    if table is not None:
        dt = o._by_bucket(ds, found, table)
        res["dtable"] = dt, u * dt.abs() + tiny + o._by_bucket(off, found, table)
    return res
