"""Plain 64-bit forms of the encoder operators, written from their definitions, and
bounds on what a kernel may be off that rounds where it has to.

U is the unit roundoff of the results' type: a value rounded once is off by at most U of
itself.  Each bound adds to that what the operands' roundings inside a kernel (the
probabilities and ds, as the matrix cores take them, and the saved output) do to
the result, term by term with absolute values, and small change for fp32 sums.
"""

from __future__ import annotations

import math

import torch

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half the spacing of subnormals
F32 = 2.0**-24


def within(got, want, bound, what):
    """Every value of ``got`` is within ``bound`` of ``want`` (infinities and NaN alike in both)."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, not {tuple(want.shape)}"
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = odd & ~torch.isnan(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities in other places"
    off = (got - want).abs() - bound
    off[odd] = -1.0
    if off.numel():
        at = int(off.argmax())
        assert float(off.max()) <= 0, (f"{what}: {got.reshape(-1)[at]} instead of {want.reshape(-1)[at]}, "
                                       f"{float((got - want).abs().reshape(-1)[at] / bound.expand_as(want).reshape(-1)[at]):.2f} "
                                       "of the bound")


# ---- layer norm -------------------------------------------------------------------


def norm(x, w, b, eps):
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    y = (x - mean) * rstd * w
    return (y if b is None else y + b), mean[..., 0], rstd[..., 0]


def norm_bounds(x, w, b, eps, dtype):
    """Bounds of y, mean, rstd: the mean is off by a few fp32 roundings of the row's magnitude."""
    y, mean, rstd = norm(x, w, b, eps)
    slip = 16 * F32 * x.abs().amax(-1)
    xhat = (x - mean[..., None]) * rstd[..., None]
    xslip = slip * rstd + 16 * F32
    y_bound = U[dtype] * y.abs() + TINY[dtype] + (1 + xhat.abs()) * xslip[..., None] * w.abs() + 4 * F32 * (y.abs() + (0 if b is None else b.abs()))
    return y_bound, slip, rstd * (16 * F32 + 2 * slip * rstd)


def _columns(t):
    return t.reshape(-1, t.shape[-1]).sum(0)


def norm_grads(dy, x, w, mean, rstd):
    xhat = (x - mean[..., None]) * rstd[..., None]
    g = dy * w
    dx = rstd[..., None] * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx, _columns(dy * xhat), _columns(dy)


def norm_grad_bounds(dy, x, w, mean, rstd, dtype):
    dx, dw, db = norm_grads(dy, x, w, mean, rstd)
    xhat = (x - mean[..., None]) * rstd[..., None]
    g = (dy * w).abs()
    sizes = g + g.mean(-1, keepdim=True) + xhat.abs() * (g * xhat.abs()).mean(-1, keepdim=True)
    # (x - mean) rounds relative to x; sums of up to a few hundred terms in a row
    slip = 16 * F32 * (1 + x.abs().amax(-1, keepdim=True) * rstd[..., None])
    n = max(1, x.numel() // x.shape[-1])
    chain = F32 * (16 + math.sqrt(n))
    return (U[dtype] * dx.abs() + TINY[dtype] + 2 * slip * rstd[..., None] * sizes * (1 + xhat.abs()),
            U[dtype] * dw.abs() + TINY[dtype] + chain * _columns((dy * xhat).abs()) + _columns(dy.abs() * slip),
            U[dtype] * db.abs() + TINY[dtype] + chain * _columns(dy.abs()))


# ---- linear -------------------------------------------------------------------------


def activate(z, act):
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    if act == "relu":
        return z.clamp(min=0)
    return torch.tanh(z) if act == "tanh" else z


def slope(z, act):
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "relu":
        return (z > 0).to(z.dtype)
    return torch.cosh(z).pow(-2) if act == "tanh" else torch.ones_like(z)


def linear(x, w, b, act, res):
    z = x @ w.T
    if b is not None:
        z = z + b
    y = activate(z, act)
    return (y if res is None else y + res), z


def linear_bounds(x, w, b, act, res, dtype):
    """The sum's fp32 roundings (any order of k terms), an activation of slope at most 1.13 that is good to 1e-6, a rounding."""
    y, z = linear(x, w, b, act, res)
    size = x.abs() @ w.abs().T + (0 if b is None else b.abs())
    slip = F32 * (8 + math.sqrt(x.shape[-1])) * size
    return (U[dtype] * y.abs() + TINY[dtype] + 1.13 * slip + 1e-6 * (1 + activate(z, act).abs()) + 2 * F32 * y.abs(),
            U[dtype] * z.abs() + TINY[dtype] + slip)


def linear_grads(dy, x, w, act, pre):
    dz = dy if act is None else dy * slope(pre, act)
    return dz @ w, dz.reshape(-1, dz.shape[-1]).T @ x.reshape(-1, x.shape[-1]), dz.reshape(-1, dz.shape[-1]).sum(0)


def linear_grad_bounds(dy, x, w, act, pre, dtype):
    dx, dw, db = linear_grads(dy, x, w, act, pre)
    dz = dy if act is None else dy * slope(pre, act)
    u = U[dtype]
    inner = 0.0 if act is None else u  # dz is rounded before the products
    eps = (0 if act is None else 2e-6) * dy.abs() + (0 if act is None else TINY[dtype])
    off = inner * dz.abs() + eps
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    m = flat(x).shape[0]
    chain_x, chain_w = F32 * (8 + math.sqrt(w.shape[0])), F32 * (8 + math.sqrt(m))
    size_x = dz.abs() @ w.abs()
    size_w = flat(dz).abs().T @ flat(x).abs()
    return (u * dx.abs() + TINY[dtype] + off @ w.abs() + chain_x * size_x,
            u * dw.abs() + TINY[dtype] + flat(off).T @ flat(x).abs() + chain_w * size_w,
            u * db.abs() + TINY[dtype] + flat(eps).sum(0) + chain_w * flat(dz).abs().sum(0))


# ---- attention -----------------------------------------------------------------------


def bucket(rel, buckets, causal, max_distance):
    """By counting boundaries: distance n is past boundary t when (n / exact)^wide >= (max_distance / exact)^t,
    in whole numbers n^wide exact^t >= max_distance^t exact^wide."""
    one = buckets if causal else buckets // 2
    exact = one // 2
    wide = one - exact

    def of(n):
        if n < exact:
            return n
        return exact + sum(n**wide * exact**t >= max_distance**t * exact**wide for t in range(1, wide))

    def at(r):
        r = int(r)
        if causal:
            return of(max(-r, 0))
        return of(-r) if r <= 0 else one + of(r)

    known = {int(r): at(r) for r in rel.unique()}
    return rel.clone().apply_(lambda r: known[int(r)])


def attention_parts(q, k, v, scale, table=None, max_distance=128, causal=False, key_lengths=None, query_lengths=None,
                    query_start=None):
    """(scores [b, h, lq, lk] with -inf where masked, probabilities, log sums, found buckets [b, lq, lk] or None)."""
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    kk, vv = (t.repeat_interleave(h // hk, 2) for t in (k, v))
    start = torch.full((b,), lk - lq) if query_start is None else query_start.long().cpu()
    rel = torch.arange(lk)[None, None, :] - torch.arange(lq)[None, :, None] - start[:, None, None]
    seen = torch.ones(b, lq, lk, dtype=torch.bool)
    if causal:
        seen &= rel <= 0
    if key_lengths is not None:
        seen &= (torch.arange(lk)[None, :] < key_lengths.long().cpu()[:, None])[:, None, :]
    if query_lengths is not None:
        seen &= (torch.arange(lq)[None, :] < query_lengths.long().cpu()[:, None])[:, :, None]
    kk = torch.where(seen.any(1)[:, :, None, None], kk, torch.zeros_like(kk))  # what lies in keys nobody sees is nobody's
    vv = torch.where(seen.any(1)[:, :, None, None], vv, torch.zeros_like(vv))
    qq = torch.where(seen.any(2)[:, :, None, None], q, torch.zeros_like(q))
    s = torch.matmul(qq.transpose(1, 2), kk.permute(0, 2, 3, 1)) * scale
    found = None
    if table is not None:
        found = bucket(rel, table.shape[0], causal, max_distance)
        s = s + table[found].permute(0, 3, 1, 2)
    s = s.masked_fill(~seen[:, None], -math.inf)
    lse = torch.logsumexp(s, 3)
    p = torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None])
    return s, p, lse, found, qq, kk, vv


def attention(q, k, v, scale, **more):
    _, p, lse, _, _, _, vv = attention_parts(q, k, v, scale, **more)
    return torch.matmul(p, vv.transpose(1, 2)).transpose(1, 2), lse


SCORE = 2.0**-16  # a probability's relative error from fp32 scores up to some tens, exponentials and sums


def attention_bounds(q, k, v, scale, dtype, **more):
    s, p, lse, _, _, _, vv = attention_parts(q, k, v, scale, **more)
    out = torch.matmul(p, vv.transpose(1, 2)).transpose(1, 2)
    size = torch.matmul(p, vv.transpose(1, 2).abs()).transpose(1, 2)
    lowest = TINY[dtype] * vv.abs().sum(1, keepdim=True)  # probabilities (relative to the largest) that are subnormal
    return (U[dtype] * out.abs() + TINY[dtype] + (U[dtype] + SCORE) * size + lowest,
            torch.full_like(lse, 2.0**-17) + 2.0**-20 * torch.where(torch.isinf(lse), torch.zeros_like(lse), lse).abs())


def _share(t, hk):
    b, l, h, d = t.shape
    return t.reshape(b, l, hk, h // hk, d).sum(3)


def attention_grads(do, q, k, v, scale, table=None, **more):
    """(dq, dk, dv, dtable or None) by the formulas."""
    _, p, _, found, qq, kk, vv = attention_parts(q, k, v, scale, table, **more)
    seen_rows = (p.sum(3) > 0)[..., None]
    g = do.transpose(1, 2)
    g = torch.where(seen_rows, g, torch.zeros_like(g))
    qt, kt, vt = (t.transpose(1, 2) for t in (qq, kk, vv))
    dp = torch.matmul(g, vt.transpose(2, 3).contiguous())
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    dq = torch.matmul(ds, kt).transpose(1, 2) * scale
    dk = _share(torch.matmul(ds.transpose(2, 3).contiguous(), qt).transpose(1, 2), k.shape[2]) * scale
    dv = _share(torch.matmul(p.transpose(2, 3).contiguous(), g).transpose(1, 2), k.shape[2])
    return dq, dk, dv, None if table is None else _by_bucket(ds, found, table)


def _by_bucket(pairs, found, table):
    out = torch.zeros_like(table)
    for h in range(table.shape[1]):
        out[:, h] = torch.bincount(found.reshape(-1), pairs[:, h].reshape(-1), table.shape[0])
    return out


def attention_grad_bounds(do, q, k, v, scale, dtype, table=None, **more):
    """delta is taken from the rounded output, off by U sum |do out|."""
    u, tiny = U[dtype], TINY[dtype]
    dq, dk, dv, dt = attention_grads(do, q, k, v, scale, table, **more)
    _, p, _, found, qq, kk, vv = attention_parts(q, k, v, scale, table, **more)
    g = do.transpose(1, 2)
    g = torch.where((p.sum(3) > 0)[..., None], g, torch.zeros_like(g))
    qt, kt, vt = (t.transpose(1, 2) for t in (qq, kk, vv))
    out = torch.matmul(p, vt)
    slip = u * (g * out).abs().sum(3, keepdim=True) + tiny * g.abs().sum(3, keepdim=True)
    size = torch.matmul(g.abs(), vt.abs().transpose(2, 3).contiguous())
    dp = torch.matmul(g, vt.transpose(2, 3).contiguous())
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    off = SCORE * ds.abs() + p * (slip + 2.0**-20 * size)      # of ds, before it is rounded
    round_p, round_ds = u * p + tiny, u * ds.abs() + tiny
    hk = k.shape[2]
    bq = u * dq.abs() + tiny + scale * torch.matmul(off + round_ds, kt.abs()).transpose(1, 2)
    bk = u * dk.abs() + tiny + scale * _share(torch.matmul((off + round_ds).transpose(2, 3).contiguous(), qt.abs()).transpose(1, 2), hk)
    bv = u * dv.abs() + tiny + _share(torch.matmul((SCORE * p + round_p).transpose(2, 3).contiguous(), g.abs()).transpose(1, 2), hk)
    bt = None if dt is None else u * dt.abs() + tiny + _by_bucket(off, found, table)
    return bq, bk, bv, bt
