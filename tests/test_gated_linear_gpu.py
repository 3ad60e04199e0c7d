"""The gated feed-forward block against its 64-bit plain form (needs an MI355X).

No counterpart in the reference.  Bounds are derived in long_encoder_oracle and encoder_oracle.
"""

from __future__ import annotations

import math

import pytest
import torch

import encoder_oracle as o
import long_encoder_oracle as lo
from cuda_vector_search import encoder
from test_encoder_gpu import rand, say

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
NAMES = ("dx", "dgate", "dup", "dgate_bias", "dup_bias")

# sizes that take each tile, whole and in parts, in each of the products
SIZES = [(1, 8, 8, "silu", F16), (23, 384, 1536, "gelu", F16), (65, 72, 136, "sigmoid", BF16), (64, 64, 64, None, F16),
         (300, 768, 104, "tanh", F16), (257, 200, 520, "relu", BF16), (7, 2048, 768, "silu", BF16), (2049, 264, 1000, "silu", F16),
         (416, 2328, 408, "gelu", BF16), (404, 3728, 616, "silu", F16), (4500, 640, 1160, "gelu", BF16), (6478, 64, 1752, "silu", F16),
         (5956, 1976, 64, "tanh", BF16)]


def inputs(m, k, n, dtype, seed=61):
    x = rand((m, k), seed, dtype)
    wg, wu = rand((n, k), seed + 1, dtype, 1 / math.sqrt(k)), rand((n, k), seed + 2, dtype, 1 / math.sqrt(k))
    bg, bu = rand((n,), seed + 3, dtype, 0.3), rand((n,), seed + 4, dtype, 0.3)
    return x, wg, wu, bg, bu, rand((m, n), seed + 5, dtype, 0.5)


@pytest.mark.parametrize("m,k,n,act,dtype", SIZES)
def test_gated_linear(eng, m, k, n, act, dtype):
    say("gated", m, k, n, act, dtype)
    (x, xd), (wg, wgd), (wu, wud), (bg, bgd), (bu, bud), (dy, dyd) = inputs(m, k, n, dtype)
    y, pre = encoder.gated_linear_forward(x, wg, wu, bg, bu, act, keep_pre=True)
    args = (xd, wgd, wud, bgd, bud, act)
    for name, a, r, t in zip(("y", "pre"), (y, pre), lo.gated(*args), lo.gated_bounds(*args, dtype)):
        o.within(a, r, t, name)
    args = (xd, wgd, wud, None, bud, act)
    o.within(encoder.gated_linear(x, wg, wu, None, bu, act), lo.gated(*args)[0], lo.gated_bounds(*args, dtype)[0], "y without a bias")
    args = (dyd, xd, wgd, wud, pre.double().cpu(), act)
    grads = encoder.gated_linear_backward(dy, x, wg, wu, pre, act)
    for name, a, r, t in zip(NAMES, grads, lo.gated_grads(*args), lo.gated_grad_bounds(*args, dtype)):
        o.within(a, r, t, name)
    again = encoder.gated_linear_backward(dy, x, wg, wu, pre, act)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    for needs in ((False, True, False, True, False), (False, False, True, False, True), (True, False, False, False, False),
                  (False,) * 5):
        some = encoder.gated_linear_backward(dy, x, wg, wu, pre, act, needs)
        for name, need, a, r, t in zip(NAMES, needs, some, lo.gated_grads(*args), lo.gated_grad_bounds(*args, dtype)):
            if need:
                o.within(a, r, t, name + " alone")
            else:
                assert a is None


# A value rounded once is off by at most U relative to it, evenly: a tensor so rounded by at most U / sqrt(3) of its norm (5
# standard deviations of a mean of 1000 squares, sqrt(0.8 / 1000) each, give 1.07).  Up to 32 rows nothing else is
# rounded to 16 bits (fp16's subnormals and fp32 sums are below a hundredth of it here); of more rows dz is.
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,k,n,act", [(1, 1024, 384, "silu"), (2, 1000, 64, "sigmoid"), (6, 1536, 8, "relu"), (8, 1000, 4096, "tanh"),
                                       (32, 384, 200, "gelu"), (33, 384, 200, None), (3, 8192, 16, "silu")])
def test_gated_gradients_errors_are_the_roundings(eng, dtype, m, k, n, act):
    say("gated errors", m, k, n, act, dtype)
    (x, xd), (wg, wgd), (wu, wud), (bg, _), (bu, _), (dy, dyd) = inputs(m, k, n, dtype, seed=67)
    _, pre = encoder.gated_linear_forward(x, wg, wu, bg, bu, act, keep_pre=True)
    want = lo.gated_grads(dyd, xd, wgd, wud, pre.double().cpu(), act)
    for name, a, r in list(zip(NAMES, encoder.gated_linear_backward(dy, x, wg, wu, pre, act), want))[:3]:
        off = float((a.double().cpu() - r).norm() / r.norm())
        assert off <= 1.08 * o.U[dtype] * math.sqrt((1 if m <= 32 else 2) / 3), (name, off / o.U[dtype])


def test_gated_gradients_past_the_type(eng):
    """Of few rows too, what rounding makes infinite stays so, and NaN reaches its own rows' results only."""
    x, g, u = (torch.ones(s, dtype=F16, device="cuda") for s in ((2, 16), (8, 16), (8, 16)))
    pre = torch.full((2, 16), 300.0, dtype=F16, device="cuda")
    dy = torch.full((2, 8), 300.0, dtype=F16, device="cuda")
    dx = encoder.gated_linear_backward(dy, x, g, u, pre, None)[0]
    assert torch.isposinf(dx).all()
    dy[1] = math.nan
    dx, dg, du = encoder.gated_linear_backward(dy, x, g, u, pre, None)[:3]
    assert torch.isposinf(dx[0]).all() and dx[1].isnan().all() and dg.isnan().all() and du.isnan().all()


def test_gated_linear_halves_of_one_weight_and_shapes(eng):
    """Weights that are halves of one, or stored the other way; rows that are views."""
    big, bigd = rand((6, 40, 600), 16, F16)
    both, bothd = rand((144, 200), 17, F16, 0.1)
    (wg, wu), (wgd, wud) = both.chunk(2), bothd.chunk(2)
    for view in (lambda t: t[:, :, 104:304], lambda t: t[:, 2, 1:201], lambda t: t[:, :, :400:2], lambda t: t[3:4, :, 8:208],
                 lambda t: t[:, :1, 8:208].expand(6, 4, 200), lambda t: t[0, 0, :200]):
        x, xd = view(big), view(bigd)
        y, pre = encoder.gated_linear_forward(x, wg, wu, keep_pre=True)
        o.within(y, lo.gated(xd, wgd, wud, None, None, "silu")[0], lo.gated_bounds(xd, wgd, wud, None, None, "silu", F16)[0], "y")
        dy = (y * 0.5)[..., :72]
        args = (dy.double().cpu(), xd, wgd, wud, pre.double().cpu(), "silu")
        for name, a, r, t in zip(NAMES, encoder.gated_linear_backward(dy, x, wg, wu, pre), lo.gated_grads(*args), lo.gated_grad_bounds(*args, F16)):
            o.within(a, r, t, name + " of a view")
    x = big[:, :, :200]
    turned = wg.t().contiguous().t()
    assert torch.equal(encoder.gated_linear(x, turned, wu), encoder.gated_linear(x, wg, wu))


def test_gated_linear_reads_nothing_outside(eng):
    """NaN on every side of the operands changes nothing."""
    m, k, n = 77, 136, 200

    def framed(rows, cols):
        field = torch.full((rows + 2, cols + 16), math.nan, device="cuda", dtype=BF16)
        field[1:-1, 8:-8] = torch.randn(rows, cols, device="cuda").to(BF16)
        return field[1:-1, 8:-8]

    x, dy = framed(m, k), framed(m, n)
    wg, wu = framed(3 * n, k)[:n].contiguous(), torch.randn(n, k, device="cuda").to(BF16)
    y, pre = encoder.gated_linear_forward(x, wg, wu, keep_pre=True)
    assert torch.isfinite(y).all() and torch.equal(y, encoder.gated_linear(x.contiguous(), wg, wu))
    for a, b in zip(encoder.gated_linear_backward(dy, x, wg, wu, pre),
                    encoder.gated_linear_backward(dy.contiguous(), x.contiguous(), wg, wu, pre)):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_gated_linear_empty(eng):
    x = torch.empty(0, 16, device="cuda", dtype=F16)
    w = torch.randn(24, 16, device="cuda").to(F16)
    y, pre = encoder.gated_linear_forward(x, w, w, keep_pre=True)
    assert y.shape == (0, 24) and pre.shape == (0, 48)
    grads = encoder.gated_linear_backward(y, x, w, w, pre)
    assert grads[0].shape == (0, 16) and grads[1].shape == (24, 16)
    assert not any(g.any() for g in grads[1:])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("act", ["silu", "sigmoid", "gelu", "relu", "tanh", None])
def test_gated_linear_tails(eng, act, dtype):
    """Gates far out on both sides, small and large factors: forward, and both factors' gradients."""
    z = torch.tensor([-60000.0, -88.0, -30.0, -9.0, -5.5, -3.0, -1.2785, -0.01, -1e-5, 0.0, 1e-5, 0.01, 3.0, 9.0, 30.0, 60000.0])
    eye = torch.eye(16, dtype=dtype, device="cuda")
    g = z.to(dtype)
    zero = torch.zeros(16, 16, dtype=dtype)
    x = torch.zeros(16, 16, dtype=dtype)
    for u in (1.0, -0.001, 0.25):
        up = torch.full((16,), u).to(dtype)
        gd, ud = g.double(), up.double()
        y = encoder.gated_linear(x.cuda(), eye, zero.cuda(), g.cuda(), up.cuda(), act)
        want = (lo.activate(gd, act) * ud).expand(16, 16)
        size = lo.activate(gd, act).abs().expand(16, 16)
        o.within(y, want, o.U[dtype] * want.abs() + o.TINY[dtype] + 1e-6 * (1 + size) * ud.abs() + 2 * o.F32 * want.abs(), f"{act} times {u}")
        pre = torch.cat([g, up]).expand(16, 32).cuda()
        dy = torch.full((16, 16), 0.5, dtype=dtype, device="cuda")
        grads = encoder.gated_linear_backward(dy, eye, eye, eye, pre, act)
        args = (dy.double().cpu(), eye.double().cpu(), eye.double().cpu(), eye.double().cpu(), pre.double().cpu(), act)
        for name, a, r, t in zip(NAMES, grads, lo.gated_grads(*args), lo.gated_grad_bounds(*args, dtype)):
            finite = r.abs() < torch.finfo(dtype).max
            o.within(torch.where(finite.cuda(), a, torch.zeros_like(a)), torch.where(finite, r, torch.zeros_like(r)), t, f"{name}, {act}")


def test_gated_linear_overflow_and_nan_stay_in_their_rows(eng):
    x = torch.randn(200, 64, device="cuda").to(F16)
    w, v = (torch.randn(72, 64, device="cuda").to(F16) for _ in range(2))
    want = encoder.gated_linear(x, w, v)
    bad = x.clone()
    bad[3, 5], bad[130, 0], bad[77] = math.nan, math.inf, 60000.0
    y = encoder.gated_linear(bad, w, v)
    rows = torch.ones(200, dtype=torch.bool)
    rows[[3, 130, 77]] = False
    assert torch.equal(y[rows], want[rows]) and torch.isnan(y[3]).all() and not torch.isfinite(y[130]).any()


def test_gated_linear_through_autograd_and_against_differences(eng):
    """The block as a model has it, up, gate and down, with halves of one weight: the gradients'
    product with a direction is the change of the 64-bit forward along it."""
    torch.manual_seed(6)
    t = {n: (torch.randn(*s) * c).to(BF16) for n, s, c in (
        ("x", (3, 29, 32), 1.0), ("w", (96, 32), 0.25), ("b", (48,), 0.2), ("down", (32, 48), 0.2))}
    weight = torch.randn(3, 29, 32).to(BF16)

    def ours(p):
        gate, up = p["w"].chunk(2)
        return encoder.linear(encoder.gated_linear(p["x"], gate, up, p["b"]), p["down"], residual=p["x"])

    def plain(p):
        gate, up = p["w"].chunk(2)
        return lo.gated(p["x"], gate, up, p["b"], None, "silu")[0] @ p["down"].T + p["x"]

    dev = {n: v.cuda().requires_grad_() for n, v in t.items()}
    (ours(dev) * weight.cuda()).float().sum().backward()
    base = {n: v.double() for n, v in t.items()}
    for n in t:
        step = torch.randn(t[n].shape, dtype=torch.float64)
        eps = 1e-5
        change = [(plain({**base, n: base[n] + s * eps * step}) * weight.double()).sum() for s in (1, -1)]
        want = float(change[0] - change[1]) / (2 * eps)
        got = float((dev[n].grad.double().cpu() * step).sum())
        room = 8 * o.U[BF16] * float(dev[n].grad.double().norm())  # each of the chain's roundings gives a few U of the gradient's norm
        assert abs(got - want) <= room, f"{n}: {got}, {want} by differences, {room}"


def test_gated_linear_frozen_weights(eng):
    x = torch.randn(9, 16, device="cuda").to(F16).requires_grad_()
    w, v = (torch.randn(24, 16, device="cuda").to(F16) for _ in range(2))
    v.requires_grad_()
    encoder.gated_linear(x, w, v).float().sum().backward()
    assert w.grad is None and v.grad.shape == v.shape and x.grad.shape == x.shape
    with torch.no_grad():
        assert not encoder.gated_linear(x, w, v).requires_grad
    v.grad.add_(1)  # (a gradient that shares memory with none)


def test_gated_linear_refusals(eng):
    def t(*shape, dtype=F16):
        return torch.randn(*shape, device="cuda").to(dtype)

    x, w, pre = t(4, 16), t(24, 16), t(4, 48)
    for call, reason in (
        (lambda: encoder.gated_linear(x.float(), w.float(), w.float()), "bfloat16"),
        (lambda: encoder.gated_linear(x, w, t(16, 16)), "up must have shape"),
        (lambda: encoder.gated_linear(x, t(24, 24), w), "as wide"),
        (lambda: encoder.gated_linear(x, t(12, 16), t(12, 16)), "multiples of 8"),
        (lambda: encoder.gated_linear(x, w, w.to(BF16)), "type"),
        (lambda: encoder.gated_linear(x, w, w.cpu()), "CUDA"),
        (lambda: encoder.gated_linear(x, w, w, t(16)), "gate_bias"),
        (lambda: encoder.gated_linear(x, w, w, None, t(24).to(BF16)), "type"),
        (lambda: encoder.gated_linear_backward(t(4, 16), x, w, w, pre), "dy"),
        (lambda: encoder.gated_linear_backward(t(4, 24), x, w, w, t(4, 24)), "pre"),
    ):
        with pytest.raises(RuntimeError, match=reason):
            call()
    with pytest.raises(ValueError, match="activation"):
        encoder.gated_linear(x, w, w, activation="swish")
