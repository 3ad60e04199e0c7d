"""The text-encoder operators against 64-bit plain forms (needs an MI355X).

No counterpart in the reference.  Each result is held to a bound derived in
encoder_oracle from where a kernel has to round, at the sizes and masks where
one can go wrong; gradients are held to the formulas' and to differences of the
64-bit forward.
"""

from __future__ import annotations

import math

import pytest
import torch

import encoder_oracle as o
from cuda_vector_search import encoder

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def say(*a):
    print(*a, flush=True)


def rand(shape, seed, dtype, scale=1.0, shift=0.0):
    """(GPU tensor, its values in 64 bits on the CPU)."""
    g = torch.Generator().manual_seed(seed)
    t = (torch.randn(shape, generator=g) * scale + shift).to(dtype)
    return t.cuda(), t.double()


# ---- layer norm ---------------------------------------------------------------------

NORM = [(1, 8, F16), (3, 384, F16), (5, 33, F16), (130, 768, BF16), (2, 1, F32), (7, 1000, F32), (4, 2048, BF16),
        (9, 2047, F16), (3, 2056, BF16), (2, 5001, F32), (1031, 136, F32), (2500, 24, F16), (65, 520, F32)]


@pytest.mark.parametrize("rows,width,dtype", NORM)
def test_layer_norm(eng, rows, width, dtype):
    say("norm", rows, width, dtype)
    x, xd = rand((rows, width), 1, dtype, 2.0, 0.7)
    w, wd = rand((width,), 2, dtype, 0.3, 1.0)
    b, bd = rand((width,), 3, dtype)
    dy, dyd = rand((rows, width), 4, dtype, 0.5)
    got = encoder.layer_norm_forward(x, w, b, 1e-5)
    for name, a, r, t in zip(("y", "mean", "rstd"), got, o.norm(xd, wd, bd, 1e-5), o.norm_bounds(xd, wd, bd, 1e-5, dtype)):
        o.within(a, r, t, name)
    plain = encoder.layer_norm(x, w, None, 1e-5)
    o.within(plain, o.norm(xd, wd, None, 1e-5)[0], o.norm_bounds(xd, wd, None, 1e-5, dtype)[0], "y without bias")
    mean, rstd = got[1].double().cpu(), got[2].double().cpu()
    grads = encoder.layer_norm_backward(dy, x, w, got[1], got[2])
    for name, a, r, t in zip(("dx", "dweight", "dbias"), grads, o.norm_grads(dyd, xd, wd, mean, rstd),
                             o.norm_grad_bounds(dyd, xd, wd, mean, rstd, dtype)):
        o.within(a, r, t, name)
    again = encoder.layer_norm_backward(dy, x, w, got[1], got[2])
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


def test_layer_norm_strides_offsets_and_shapes(eng):
    big, bigd = rand((6, 5, 900), 5, F16)
    w, wd = rand((384,), 6, F16)
    for view in (lambda t: t[:, :, 100:484], lambda t: t[:, 2, 1:385], lambda t: t[:, :, :768:2], lambda t: t[3:4, :, 7:391],
                 lambda t: t[:, :1, 8:392].expand(6, 4, 384), lambda t: t[0, 0, :384]):
        x, xd = view(big), view(bigd)
        y, mean, rstd = encoder.layer_norm_forward(x, w, None)
        o.within(y, o.norm(xd, wd, None, 1e-5)[0], o.norm_bounds(xd, wd, None, 1e-5, F16)[0], "y")
        dx, dw, db = encoder.layer_norm_backward(x, x, w, mean, rstd)
        args = (xd, xd, wd, mean.double().cpu(), rstd.double().cpu())
        for a, r, t in zip((dx, dw, db), o.norm_grads(*args), o.norm_grad_bounds(*args, F16)):
            o.within(a, r, t, "gradient of a view")


def test_layer_norm_empty_and_odd_values(eng):
    w = torch.ones(64, device="cuda", dtype=F16)
    x = torch.empty(0, 64, device="cuda", dtype=F16)
    y, mean, rstd = encoder.layer_norm_forward(x, w, w)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = encoder.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    x = torch.randn(4, 64, device="cuda").to(F16)
    x[1] = 3.0             # no variance: only eps
    x[2, 5] = math.inf
    x[3, 6] = math.nan
    y = encoder.layer_norm(x, w)
    assert torch.isfinite(y[0]).all() and torch.equal(y[1], torch.zeros_like(y[1]))
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()


# ---- linear --------------------------------------------------------------------------

LINEAR = [(1, 8, 8, None, F16), (23, 384, 1536, "gelu", F16), (64, 64, 64, "relu", BF16), (65, 72, 136, "tanh", F16),
          (300, 768, 104, "gelu", BF16), (129, 200, 520, None, F16), (1000, 384, 384, "gelu", F16), (7, 2048, 768, None, BF16),
          (2049, 264, 1000, "gelu", BF16), (4100, 128, 1032, None, F16), (4500, 640, 1160, "relu", BF16),
          # sizes whose products take the larger tiles, whole and in parts
          (6478, 64, 1752, "gelu", BF16), (5956, 1976, 64, "tanh", F16), (404, 3728, 3240, None, BF16), (8303, 2440, 392, "gelu", F16),
          (8486, 64, 912, "tanh", F16), (6669, 1192, 64, "gelu", BF16), (416, 2328, 3408, "relu", F16), (6171, 520, 3296, None, F16)]


@pytest.mark.parametrize("m,k,n,act,dtype", LINEAR)
def test_linear(eng, m, k, n, act, dtype):
    say("linear", m, k, n, act, dtype)
    x, xd = rand((m, k), 11, dtype)
    w, wd = rand((n, k), 12, dtype, 1 / math.sqrt(k))
    b, bd = rand((n,), 13, dtype, 0.3)
    res, rd = rand((m, n), 14, dtype)
    dy, dyd = rand((m, n), 15, dtype, 0.5)
    y, pre = encoder.linear_forward(x, w, b, act, res, keep_pre=True)
    want, bounds = o.linear(xd, wd, bd, act, rd), o.linear_bounds(xd, wd, bd, act, rd, dtype)
    o.within(y, want[0], bounds[0], "y")
    o.within(pre, want[1], bounds[1], "pre")
    bare = encoder.linear(x, w, activation=act)
    o.within(bare, o.linear(xd, wd, None, act, None)[0], o.linear_bounds(xd, wd, None, act, None, dtype)[0], "y without bias and residual")
    pd = pre.double().cpu()
    grads = encoder.linear_backward(dy, x, w, act, pre)
    for name, a, r, t in zip(("dx", "dweight", "dbias"), grads, o.linear_grads(dyd, xd, wd, act, pd),
                             o.linear_grad_bounds(dyd, xd, wd, act, pd, dtype)):
        o.within(a, r, t, name)
    again = encoder.linear_backward(dy, x, w, act, pre)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    assert encoder.linear_backward(dy, x, w, act, pre, (False, True, False))[::2] == (None, None)


def test_linear_strides_offsets_and_shapes(eng):
    big, bigd = rand((6, 40, 600), 16, F16)
    w, wd = rand((72, 200), 17, F16, 0.1)
    for view in (lambda t: t[:, :, 104:304], lambda t: t[:, 2, 1:201], lambda t: t[:, :, :400:2], lambda t: t[3:4, :, 8:208],
                 lambda t: t[:, :1, 8:208].expand(6, 4, 200), lambda t: t[0, 0, :200]):
        x, xd = view(big), view(bigd)
        y, pre = encoder.linear_forward(x, w, activation="gelu", keep_pre=True)
        o.within(y, o.linear(xd, wd, None, "gelu", None)[0], o.linear_bounds(xd, wd, None, "gelu", None, F16)[0], "y")
        dy = y * 0.5
        grads = encoder.linear_backward(dy, x, w, "gelu", pre)
        args = (dy.double().cpu(), xd, wd, "gelu", pre.double().cpu())
        for a, r, t in zip(grads, o.linear_grads(*args), o.linear_grad_bounds(*args, F16)):
            o.within(a, r, t, "gradient of a view")
    wt = w.t().contiguous().t()  # a weight stored the other way
    assert torch.equal(encoder.linear(big[:, :, :200], wt), encoder.linear(big[:, :, :200], w))


def test_linear_reads_nothing_outside(eng):
    """NaN on every side of the operands changes nothing."""
    m, k, n = 77, 136, 200
    field = torch.full((m + 2, k + 16), math.nan, device="cuda", dtype=BF16)
    field[1:-1, 8:-8] = torch.randn(m, k, device="cuda").to(BF16)
    x = field[1:-1, 8:-8]
    w = torch.randn(n, k, device="cuda").to(BF16)
    dy_field = torch.full((m + 2, n + 16), math.nan, device="cuda", dtype=BF16)
    dy_field[1:-1, 8:-8] = torch.randn(m, n, device="cuda").to(BF16)
    dy = dy_field[1:-1, 8:-8]
    assert torch.equal(encoder.linear(x, w), encoder.linear(x.contiguous(), w))
    for a, b in zip(encoder.linear_backward(dy, x, w), encoder.linear_backward(dy.contiguous(), x.contiguous(), w)):
        assert torch.equal(a, b)


def test_linear_empty(eng):
    x = torch.empty(0, 16, device="cuda", dtype=F16)
    w = torch.randn(24, 16, device="cuda").to(F16)
    y, pre = encoder.linear_forward(x, w, activation="gelu", keep_pre=True)
    assert y.shape == (0, 24)
    dx, dw, db = encoder.linear_backward(y, x, w, "gelu", pre)
    assert dx.shape == (0, 16) and dw.shape == (24, 16) and not dw.any() and not db.any()


def test_linear_activation_tails(eng):
    """Values far out on both sides, infinities and NaN."""
    z = torch.tensor([-60000.0, -30.0, -9.0, -5.5, -3.0, -0.01, 0.0, 0.01, 3.0, 9.0, 30.0, 60000.0, math.inf, -math.inf, math.nan, 1.0])
    w = torch.eye(16, dtype=F16, device="cuda")
    for dtype in (F16, BF16):
        x = torch.diag(torch.nan_to_num(z, nan=0.0, posinf=0.0, neginf=0.0)).to(dtype)
        bias = torch.where(torch.isfinite(z), torch.zeros_like(z), z).to(dtype)
        xd, bd = x.double(), bias.double()
        for act in ("gelu", "relu", "tanh"):
            y = encoder.linear(x.cuda(), w.to(dtype), bias.cuda(), act)
            want, bound = o.linear(xd, torch.eye(16).double(), bd, act, None)[0], o.linear_bounds(xd, torch.eye(16).double(), torch.nan_to_num(bd, 0, 0, 0), act, None, dtype)[0]
            if act == "gelu":
                want[:, 13] = 0.0 if not torch.isnan(want[:, 13]).any() else want[:, 13]
                y[:, 13] = want[:, 13].to(y)  # minus infinity times zero: either is right
            o.within(y, want, bound, act)
            pre = torch.stack([z, z.flip(0)]).to(dtype)
            pre = torch.nan_to_num(pre, 0.0, 60000.0, -60000.0).cuda()
            dy = torch.ones(2, 16, device="cuda", dtype=dtype)
            _, _, db = encoder.linear_backward(dy, torch.ones(2, 16, device="cuda", dtype=dtype), w.to(dtype), act, pre)
            o.within(db, o.slope(torch.nan_to_num(pre.double().cpu()), act).nan_to_num(0.0).sum(0),
                     torch.full((16,), 4 * o.U[dtype] + 1e-5, dtype=torch.float64), act + " slope")


# ---- attention -----------------------------------------------------------------------

# batch, lq, lk, heads, key heads, width, type, buckets, causal, ragged
ATTENTION = [
    (1, 1, 1, 1, 1, 8, F16, 0, False, False), (1, 23, 23, 12, 12, 32, F16, 32, False, False),
    (2, 64, 64, 2, 2, 64, BF16, 32, False, False), (2, 65, 65, 2, 1, 64, F16, 32, True, False),
    (3, 130, 130, 2, 2, 40, BF16, 8, False, True), (2, 257, 257, 4, 2, 128, F16, 0, True, True),
    (1, 300, 300, 2, 2, 64, F16, 32, False, True), (2, 1, 700, 3, 3, 64, F16, 0, False, True),
    (2, 1, 333, 4, 1, 128, BF16, 16, True, False), (1, 5, 1500, 2, 2, 64, F16, 64, False, False),
    (2, 33, 100, 2, 2, 96, BF16, 0, True, True), (2, 100, 33, 2, 2, 24, F16, 32, False, False),
    (1, 513, 513, 1, 1, 32, BF16, 32, True, False), (4, 129, 31, 2, 1, 72, BF16, 0, True, False),
    (1, 400, 400, 2, 2, 16, F16, 128, False, True),
]


def attention_inputs(b, lq, lk, h, hk, d, dtype, buckets, ragged, seed=21):
    q, qd = rand((b, lq, h, d), seed, dtype, 1.5)
    k, kd = rand((b, lk, hk, d), seed + 1, dtype)
    v, vd = rand((b, lk, hk, d), seed + 2, dtype)
    do, dod = rand((b, lq, h, d), seed + 3, dtype, 0.5)
    table, td = rand((buckets, h), seed + 4, dtype) if buckets else (None, None)
    lengths = {}
    if ragged:
        g = torch.Generator().manual_seed(seed + 5)
        kl = torch.randint(0, lk + 1, (b,), generator=g).to(torch.int32)
        kl[0] = lk
        lengths["key_lengths"] = kl
        if lq == lk:
            lengths["query_lengths"] = kl
    return (q, k, v, do, table), (qd, kd, vd, dod, td), lengths


@pytest.mark.parametrize("b,lq,lk,h,hk,d,dtype,buckets,causal,ragged", ATTENTION)
def test_attention(eng, b, lq, lk, h, hk, d, dtype, buckets, causal, ragged):
    say("attention", b, lq, lk, h, hk, d, dtype, buckets, causal, ragged)
    (q, k, v, do, table), (qd, kd, vd, dod, td), lengths = attention_inputs(b, lq, lk, h, hk, d, dtype, buckets, ragged)
    for name, l in lengths.items():  # what lies past a sequence's end is nobody's business
        for n in range(b):
            for t, td_ in ((k, kd), (v, vd)) if name == "key_lengths" else ((q, qd), (do, dod)):
                t[n, int(l[n]):] = math.nan
    more = dict(causal=causal, max_distance=128, **{n: t.cuda() for n, t in lengths.items()})
    ref = dict(table=td, causal=causal, max_distance=128, **lengths)
    scale = 1 / math.sqrt(d)
    out, lse = encoder.attention_forward(q, k, v, table, **more)
    want, bounds = o.attention(qd, kd, vd, scale, **ref), o.attention_bounds(qd, kd, vd, scale, dtype, **ref)
    o.within(out, want[0], bounds[0], "out")
    o.within(lse, want[1], bounds[1], "lse")
    assert torch.equal(encoder.attention(q, k, v, table, **more), out)
    grads = encoder.attention_backward(do, q, k, v, out, lse, table, **more)
    refs = o.attention_grads(dod, qd, kd, vd, scale, **ref)
    tols = o.attention_grad_bounds(dod, qd, kd, vd, scale, dtype, **ref)
    for name, a, r, t in zip(("dq", "dk", "dv", "dtable"), grads, refs, tols):
        if r is None:
            assert a is None
        else:
            o.within(a, r, t, name)
    again = encoder.attention_backward(do, q, k, v, out, lse, table, **more)
    assert all(x is None or torch.equal(x, y) for x, y in zip(grads, again))


@pytest.mark.parametrize("lq,start", [(1, [0, 57, 199]), (4, [3, 100, 150]), (70, [-80, 0, 129]), (40, [-20, -39, 500])])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_query_start(eng, lq, start, causal):
    """Rows that stand at a position of their own in each sequence (single tokens over a
    cache of ragged length), some of which see nothing when causal."""
    (q, k, v, do, table), (qd, kd, vd, dod, td), _ = attention_inputs(3, lq, 200, 4, 2, 64, BF16, 32, False, seed=41)
    at = torch.tensor(start, dtype=torch.int32)
    kl = torch.tensor([200, 60, 199], dtype=torch.int32)
    more = dict(causal=causal, key_lengths=kl.cuda(), query_start=at.cuda(), max_distance=100)
    ref = dict(table=td, causal=causal, key_lengths=kl, query_start=at, max_distance=100)
    out, lse = encoder.attention_forward(q, k, v, table, scale=0.2, **more)
    for a, r, t in zip((out, lse), o.attention(qd, kd, vd, 0.2, **ref), o.attention_bounds(qd, kd, vd, 0.2, BF16, **ref)):
        o.within(a, r, t, "forward")
    grads = encoder.attention_backward(do, q, k, v, out, lse, table, scale=0.2, **more)
    for a, r, t in zip(grads, o.attention_grads(dod, qd, kd, vd, 0.2, **ref), o.attention_grad_bounds(dod, qd, kd, vd, 0.2, BF16, **ref)):
        o.within(a, r, t, "gradient")


@pytest.mark.parametrize("buckets,max_distance,causal", [(4, 3, False), (4, 256, True), (32, 256, False), (128, 65, True), (64, 20, False)])
def test_attention_bucket_rules(eng, buckets, max_distance, causal):
    (q, k, v, do, table), (qd, kd, vd, dod, td), _ = attention_inputs(1, 330, 330, 2, 2, 32, F16, buckets, False, seed=51)
    more = dict(causal=causal, max_distance=max_distance)
    out, lse = encoder.attention_forward(q, k, v, table, **more)
    scale = 1 / math.sqrt(32)
    o.within(out, o.attention(qd, kd, vd, scale, table=td, **more)[0], o.attention_bounds(qd, kd, vd, scale, F16, table=td, **more)[0], "out")
    grads = encoder.attention_backward(do, q, k, v, out, lse, table, **more)
    for a, r, t in zip(grads, o.attention_grads(dod, qd, kd, vd, scale, td, **more), o.attention_grad_bounds(dod, qd, kd, vd, scale, F16, td, **more)):
        o.within(a, r, t, "gradient")


def test_attention_strides_and_offsets(eng):
    """Views of one projection's output, other orders of the dimensions, expanded heads, odd offsets."""
    b, l, h, d = 2, 70, 4, 32
    qkv = torch.randn(b, l, 3, h, d, device="cuda").to(F16)
    odd = torch.randn(b * l * h * d + 1, device="cuda").to(F16)[1:].view(b, l, h, d)
    other = torch.randn(h, b, l, d, device="cuda").to(F16).permute(1, 2, 0, 3)
    one = torch.randn(b, l, 1, d, device="cuda").to(F16).expand(b, l, h, d)
    turned = torch.randn(b, l, d, h, device="cuda").to(F16).transpose(2, 3)
    for q, k, v in ((qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]), (odd, other, one), (turned, one, odd), (other, turned, qkv[:, :, 2])):
        out, lse = encoder.attention_forward(q, k, v)
        want, lsec = encoder.attention_forward(q.contiguous(), k.contiguous(), v.contiguous())
        assert torch.equal(out, want) and torch.equal(lse, lsec)
        for do in (odd, turned, one):
            a = encoder.attention_backward(do, q, k, v, out, lse)
            w = encoder.attention_backward(do.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), out, lse)
            assert all(torch.equal(x, y) for x, y in zip(a[:3], w[:3]))


def test_attention_empty(eng):
    def t(*shape):
        return torch.randn(*shape, device="cuda").to(F16)

    q, k = t(2, 5, 2, 16), t(2, 0, 2, 16)
    table = t(8, 2)
    out, lse = encoder.attention_forward(q, k, k, table, max_distance=9)
    assert not out.any() and torch.isinf(lse).all()
    dq, dk, dv, dt = encoder.attention_backward(q, q, k, k, out, lse, table, max_distance=9)
    assert not dq.any() and dk.shape == k.shape and not dt.any()
    out, lse = encoder.attention_forward(k, q, q, table, max_distance=9)
    assert out.shape == k.shape
    dq, dk, dv, dt = encoder.attention_backward(k, k, q, q, out, lse, table, max_distance=9)
    assert not dk.any() and not dv.any() and not dt.any()
    none = t(0, 5, 2, 16)
    out, lse = encoder.attention_forward(none, none, none)
    assert out.shape == none.shape
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    q = t(2, 40, 2, 16)
    out, lse = encoder.attention_forward(q, q, q, key_lengths=zero)
    assert not out.any() and (lse == -math.inf).all()
    assert not any(g.any() for g in encoder.attention_backward(q, q, q, q, out, lse, key_lengths=zero)[:3])


def test_attention_far_scores(eng):
    """Scores of some thousands, all far below or above zero, and entries of minus infinity in the table."""
    g = torch.Generator().manual_seed(3)
    q = (torch.randn(1, 50, 1, 64, generator=g) * 0.1 + 8).to(BF16)
    k = (torch.randn(1, 50, 1, 64, generator=g) * 0.1 - 8).to(BF16)
    v = torch.randn(1, 50, 1, 64, generator=g).to(BF16)
    for kk in (k, -k):
        out, lse = encoder.attention_forward(q.cuda(), kk.cuda(), v.cuda())
        want, wl = o.attention(q.double(), kk.double(), v.double(), 0.125)
        # scores near 512: fp32 holds them to 2^-15, so probabilities to about 2^-13
        o.within(out, want, 2.0**-8 * want.abs() + 2.0**-6 * torch.ones_like(want), "out")
        o.within(lse, wl, 2.0**-12 * torch.ones_like(wl), "lse")
    table = torch.zeros(8, 1, dtype=BF16)
    table[4:] = -math.inf  # nothing after the row
    table[0] = -math.inf   # nor the row itself: the first row sees nothing
    qd, kd, vd = q.double() * 0.1, k.double() * 0.1, v.double()
    q2, k2 = qd.to(BF16), kd.to(BF16)
    out, lse = encoder.attention_forward(q2.cuda(), k2.cuda(), v.cuda(), table.cuda(), max_distance=20)
    ref = dict(table=table.double(), max_distance=20)
    o.within(out, o.attention(q2.double(), k2.double(), vd, 0.125, **ref)[0], o.attention_bounds(q2.double(), k2.double(), vd, 0.125, BF16, **ref)[0], "out")
    assert not out[0, 0].any() and lse[0, 0, 0] == -math.inf
    grads = encoder.attention_backward(v.cuda(), q2.cuda(), k2.cuda(), v.cuda(), out, lse, table.cuda(), max_distance=20)
    assert all(torch.isfinite(t).all() for t in grads)


def test_attention_small_and_large_gradients_of_float16(eng):
    """Probabilities of a long uniform row and gradients at both ends of float16's range keep their digits."""
    l, d = 3000, 32
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(1, l, 1, d, generator=g).to(F16) * s for s in (0.1, 0.1, 1.0))
    out, lse = encoder.attention_forward(q.cuda(), k.cuda(), v.cuda())
    for size in (2.0**-12, 1.0, 2.0**9):
        do = (torch.randn(1, l, 1, d, generator=g) * size).to(F16)
        grads = encoder.attention_backward(do.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse)
        want = o.attention_grads(do.double(), q.double(), k.double(), v.double(), 1 / math.sqrt(d))
        for name, a, r in zip(("dq", "dk", "dv"), grads, want):
            # half the spacing of the result's subnormals, relative to its size, and a few roundings of operands
            rel = float((a.double().cpu() - r).norm() / r.norm())
            room = 2.0**-25 / float(r.square().mean().sqrt()) + 4 * 2.0**-11
            assert rel <= room, f"{name} at {size}: {rel} of {room}"


# ---- gradients against differences, and through torch's autograd ----------------------


def test_gradients_against_differences(eng):
    """The gradients' product with a direction is the change of the 64-bit forward along it."""
    torch.manual_seed(5)
    b, l, h, d, f = 2, 37, 2, 16, 32
    t = {n: (torch.randn(*s) * c).to(BF16) for n, s, c in (
        ("x", (b, l, f), 1.0), ("w", (3 * f, f), 0.3), ("b", (3 * f,), 0.1), ("table", (8, h), 1.0), ("wo", (f, f), 0.2),
        ("g", (f,), 1.0), ("c", (f,), 0.2))}
    weight = torch.randn(b, l, f).to(BF16)

    def ours(p):
        qkv = encoder.linear(p["x"], p["w"], p["b"]).view(b, l, 3, h, d)
        a = encoder.attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], p["table"], max_distance=20)
        y = encoder.linear(a.view(b, l, f), p["wo"], None, "gelu", p["x"])
        return encoder.layer_norm(y, p["g"], p["c"])

    def plain(p):
        qkv = o.linear(p["x"], p["w"], p["b"], None, None)[0].view(b, l, 3, h, d)
        a, _ = o.attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], 0.25, table=p["table"], max_distance=20)
        return o.norm(o.linear(a.reshape(b, l, f), p["wo"], None, "gelu", p["x"])[0], p["g"], p["c"], 1e-5)[0]

    dev = {n: v.cuda().requires_grad_() for n, v in t.items()}
    loss = (ours(dev) * weight.cuda()).float().sum()
    loss.backward()
    base = {n: v.double() for n, v in t.items()}
    for n in t:
        step = torch.randn(t[n].shape, dtype=torch.float64)
        eps = 1e-5
        change = [(plain({**base, n: base[n] + s * eps * step}) * weight.double()).sum() for s in (1, -1)]
        want = float(change[0] - change[1]) / (2 * eps)
        got = float((dev[n].grad.double().cpu() * step).sum())
        # a random direction's product has the gradient's norm; each of the chain's roundings gives a few U of it
        room = 10 * o.U[BF16] * float(dev[n].grad.double().norm())
        assert abs(got - want) <= room, f"{n}: {got}, {want} by differences, {room}"


def test_no_gradient_where_none_is_asked(eng):
    x = torch.randn(4, 16, device="cuda").to(F16).requires_grad_()
    w = torch.randn(16, 16, device="cuda").to(F16)
    y = encoder.layer_norm(encoder.linear(x, w, activation="relu"), w[0])
    y.sum().backward()
    assert x.grad is not None and w.grad is None
    with torch.no_grad():
        assert not encoder.linear(x, w).requires_grad


def test_other_streams_and_graph_replays(eng):
    """On a stream of the caller's own, and captured: every replay gives the eager result."""
    torch.manual_seed(9)
    x = torch.randn(3, 50, 64, device="cuda").to(F16)
    w = (torch.randn(192, 64, device="cuda") * 0.2).to(F16)
    g = torch.randn(64, device="cuda").to(F16)
    table = torch.randn(8, 4, device="cuda").to(F16)

    def step():
        n, mean, rstd = encoder.layer_norm_forward(x, g)
        qkv, _ = encoder.linear_forward(n, w)
        qkv = qkv.view(3, 50, 3, 4, 16)
        q, k, v = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
        out, lse = encoder.attention_forward(q, k, v, table, max_distance=30)
        grads = encoder.attention_backward(out, q, k, v, out, lse, table, max_distance=30)
        dqkv = torch.cat([t.reshape(3, 50, 64) for t in grads[:3]], 2)
        dn, dw, db = encoder.linear_backward(dqkv, n, w)
        return out, grads[3], dw, db, *encoder.layer_norm_backward(dn, x, g, mean, rstd)

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


# ---- refusals ---------------------------------------------------------------------------


def test_refusals(eng):
    def t(*shape, dtype=F16):
        return torch.randn(*shape, device="cuda").to(dtype)

    x = t(4, 16)
    stat = torch.zeros(4, device="cuda")
    for call, reason in (
        (lambda: encoder.layer_norm(x.double(), t(16).double()), "float32"),
        (lambda: encoder.layer_norm(x, t(8)), "shape"),
        (lambda: encoder.layer_norm(x, t(16, dtype=F32)), "type"),
        (lambda: encoder.layer_norm(x, t(16).cpu()), "CUDA"),
        (lambda: encoder.layer_norm_backward(t(3, 16), x, t(16), stat, stat), "shape"),
        (lambda: encoder.layer_norm_backward(x, x, t(16), stat[:3], stat), "mean"),
        (lambda: encoder.linear(x.float(), t(8, 16, dtype=F32)), "bfloat16"),
        (lambda: encoder.linear(x, t(8, 24)), "as wide"),
        (lambda: encoder.linear(x, t(12, 16)), "multiples of 8"),
        (lambda: encoder.linear(x, t(8, 16), t(16)), "shape"),
        (lambda: encoder.linear(x, t(8, 16), residual=t(4, 16)), "shape"),
        (lambda: encoder.linear_backward(t(4, 8), x, t(8, 16), "gelu"), "pre"),
        (lambda: encoder.attention(t(2, 3, 4, 20), t(2, 3, 4, 20), t(2, 3, 4, 20)), "multiples of 8"),
        (lambda: encoder.attention(t(2, 3, 4, 136), t(2, 3, 4, 136), t(2, 3, 4, 136)), "128"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(2, 3, 3, 16), t(2, 3, 3, 16)), "multiple of key heads"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(1, 3, 4, 16), t(1, 3, 4, 16)), "batch"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(2, 3, 4, 16), t(2, 5, 4, 16)), "must be"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(2, 3, 4, 16), t(2, 3, 4, 16), t(5, 4)), "even number"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(2, 3, 4, 16), t(2, 3, 4, 16), t(8, 3)), "buckets, heads"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(2, 3, 4, 16), t(2, 3, 4, 16), t(32, 4), max_distance=8), "max_distance"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(2, 3, 4, 16), t(2, 3, 4, 16), t(32, 4), max_distance=257), "max_distance"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(2, 3, 4, 16), t(2, 3, 4, 16), scale=0.0), "scale"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(2, 3, 4, 16), t(2, 3, 4, 16), scale=math.nan), "scale"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(2, 3, 4, 16), t(2, 3, 4, 16), key_lengths=torch.zeros(2, device="cuda")), "int32"),
        (lambda: encoder.attention(t(2, 3, 4, 16), t(2, 3, 4, 16), t(2, 3, 4, 16), key_lengths=torch.zeros(3, device="cuda", dtype=torch.int32)), "key_lengths"),
    ):
        with pytest.raises(RuntimeError, match=reason):
            call()
    with pytest.raises(ValueError, match="activation"):
        encoder.linear(x, t(8, 16), activation="swish")
