"""Bounds of attention's gradients without the slack that encoder_oracle gives where a kernel
need not lose digits: rows whose delta comes from the probabilities, and float16 operands
lifted out of the subnormals.
"""

from __future__ import annotations

import torch

import encoder_oracle as o


def grad_bounds(do, q, k, v, scale, dtype, table=None, own_delta=None, lift=0, **more):
    """Bounds of (dq, dk, dv, dtable or None), as ``encoder_oracle.attention_grad_bounds``, but:

    ``own_delta`` (bool [lq]): rows whose delta is the sum of their own p dp in fp32, so that it
    is not off by the rounding of ``out``;
    ``lift``: float16 operands are products with 2^lift (less where they would not fit: the
    largest then has 2^14 at least), so what they lose below float16's normal range is
    2^-25 of the lifted value.
    """
    u, tiny = o.U[dtype], o.TINY[dtype]
    dq, dk, dv, dt = o.attention_grads(do, q, k, v, scale, table, **more)
    _, p, _, found, qq, kk, vv = o.attention_parts(q, k, v, scale, table, **more)
    g = do.transpose(1, 2)
    g = torch.where((p.sum(3) > 0)[..., None], g, torch.zeros_like(g))
    qt, kt, vt = (t.transpose(1, 2) for t in (qq, kk, vv))
    out = torch.matmul(p, vt)
    slip = u * (g * out).abs().sum(3, keepdim=True) + tiny * g.abs().sum(3, keepdim=True)
    size = torch.matmul(g.abs(), vt.abs().transpose(2, 3).contiguous())
    if own_delta is not None:
        exact = 2.0**-20 * (p * size).sum(3, keepdim=True)
        slip = torch.where(own_delta[None, None, :, None], exact, slip)
    dp = torch.matmul(g, vt.transpose(2, 3).contiguous())
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    off = o.SCORE * ds.abs() + p * (slip + 2.0**-20 * size)
    low = tiny * 2.0**-lift
    # a row's (for dq) or a key's (for dk, over the query heads) largest value, where 2^lift leaves no room for it
    round_q = u * ds.abs() + low * (1 + ds.abs().amax(3, keepdim=True))
    round_k = u * ds.abs() + low * (1 + ds.abs().amax((1, 2), keepdim=True))
    round_p = u * p + low
    hk = k.shape[2]
    bq = u * dq.abs() + tiny + scale * torch.matmul(off + round_q, kt.abs()).transpose(1, 2)
    bk = u * dk.abs() + tiny + scale * o._share(torch.matmul((off + round_k).transpose(2, 3).contiguous(), qt.abs()).transpose(1, 2), hk)
    bv = u * dv.abs() + tiny + o._share(torch.matmul((o.SCORE * p + round_p).transpose(2, 3).contiguous(), g.abs()).transpose(1, 2), hk)
    bt = None if dt is None else u * dt.abs() + tiny + o._by_bucket(off, found, table)
    return (dq, dk, dv, dt), (bq, bk, bv, bt)
