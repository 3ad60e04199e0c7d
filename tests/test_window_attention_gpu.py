"""Attention with a sliding window and first keys that stay visible, against its 64-bit plain form
(needs an MI355X).

No counterpart in the reference.  Bounds are derived in long_encoder_oracle and encoder_oracle.
"""

from __future__ import annotations

import math

import pytest
import torch

import encoder_oracle as o
import long_encoder_oracle as lo
from cuda_vector_search import encoder
from test_encoder_gpu import attention_inputs, say

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
GRADS = ("dq", "dk", "dv", "dtable")


def hold(tensors, doubles, scale, dtype, before, after, sinks, lengths, what="", poison=True, **more):
    """Forward and backward of the GPU tensors within the bounds; where no row sees, or is to see, NaN."""
    (q, k, v, do, table), (qd, kd, vd, dod, td) = tensors, doubles
    lengths = {n: t for n, t in lengths.items() if t is not None}
    if poison:
        _, seen = lo.window_seen(q.shape[0], q.shape[1], k.shape[1], before, after, sinks, more.get("causal", False), **lengths)
        q, k, v, do = (t.clone() for t in (q, k, v, do))
        for t in (k, v):
            t[~seen.any(1).cuda()] = math.nan
        for t in (q, do):
            t[~seen.any(2).cuda()] = math.nan
    args = dict(window=(before, after), sinks=sinks, scale=scale, **more, **{n: t.cuda() for n, t in lengths.items()})
    narrow = before + (0 if more.get("causal") else after) + min(sinks, k.shape[1]) < 64
    want = lo.window_attention(qd, kd, vd, dod, scale, dtype, before, after, sinks, td, own_delta=narrow, **more, **lengths)
    out, lse = encoder.attention_forward(q, k, v, table, **args)
    o.within(out, *want["out"], what + " out")
    o.within(lse, *want["lse"], what + " lse")
    assert torch.equal(encoder.attention(q, k, v, table, **args), out)
    grads = encoder.attention_backward(do, q, k, v, out, lse, table, **args)
    for name, a in zip(GRADS, grads):
        if name not in want:
            assert a is None
        else:
            o.within(a, *want[name], f"{what} {name}")
    again = encoder.attention_backward(do, q, k, v, out, lse, table, **args)
    assert all(a is None or torch.equal(a, b) for a, b in zip(grads, again))


# batch, lq, lk, heads, key heads, width, type, buckets, causal, ragged, before, after, sinks
CASES = [
    (1, 1, 1, 1, 1, 8, F16, 0, False, False, 0, 0, 0), (1, 23, 23, 2, 2, 32, F16, 32, False, False, 4, 4, 1),
    (2, 200, 200, 2, 2, 64, BF16, 0, False, False, 20, 20, 4), (2, 300, 300, 2, 1, 64, F16, 0, True, False, 100, 0, 4),
    (1, 700, 700, 2, 2, 64, F16, 0, False, True, 128, 128, 4), (3, 400, 400, 2, 2, 40, BF16, 32, False, True, 64, 30, 1),
    (2, 513, 513, 4, 2, 128, F16, 0, True, True, 200, 0, 16), (1, 600, 600, 4, 1, 128, BF16, 0, False, False, 90, 200, 0),
    (2, 300, 300, 2, 2, 96, BF16, 16, True, False, 33, 0, 70), (1, 400, 400, 1, 1, 16, F16, 0, False, False, 0, 3, 0),
    (2, 1, 700, 4, 1, 64, F16, 0, True, True, 100, 0, 4), (3, 1, 900, 2, 2, 128, BF16, 32, False, True, 300, 10, 0),
    (1, 5, 1500, 2, 2, 64, F16, 0, True, False, 31, 0, 200), (2, 16, 1300, 4, 2, 32, BF16, 0, True, False, 700, 0, 2),
    (2, 130, 400, 2, 2, 64, BF16, 0, True, True, 70, 0, 4), (2, 300, 90, 2, 2, 24, F16, 0, False, False, 40, 40, 3),
    (2, 300, 90, 2, 2, 64, F16, 0, False, False, 40, 40, 0), (1, 260, 260, 2, 2, 72, F16, 0, True, False, 1000, 0, 4),
    (1, 150, 150, 2, 1, 64, BF16, 64, False, False, 500, 500, 300), (2, 1100, 1100, 1, 1, 64, BF16, 0, False, False, 3, 300, 5),
]


@pytest.mark.parametrize("b,lq,lk,h,hk,d,dtype,buckets,causal,ragged,before,after,sinks", CASES)
def test_window_attention(eng, b, lq, lk, h, hk, d, dtype, buckets, causal, ragged, before, after, sinks):
    say("window", b, lq, lk, h, hk, d, dtype, buckets, causal, ragged, before, after, sinks)
    tensors, doubles, lengths = attention_inputs(b, lq, lk, h, hk, d, dtype, buckets, ragged, seed=121)
    hold(tensors, doubles, 1 / math.sqrt(d), dtype, before, after, sinks, lengths, causal=causal, max_distance=128)


# sizes whose keys are walked in parts (forward, dq) and whose rows are (dk and dv, the first keys')
PARTS = [(1, 130, 2000, 2, 2, 64, F16, 0, False, 1500, 300, 4), (1, 130, 2000, 2, 1, 128, BF16, 32, True, 1400, 0, 2),
         (1, 3000, 3000, 1, 1, 64, F16, 0, False, 1000, 500, 5), (1, 2500, 2500, 2, 1, 128, BF16, 0, True, 1100, 0, 40),
         (2, 7, 2600, 2, 2, 32, BF16, 32, False, 2000, 200, 70), (1, 1500, 1500, 2, 2, 96, F16, 16, False, 0, 20, 9)]


@pytest.mark.parametrize("b,lq,lk,h,hk,d,dtype,buckets,causal,before,after,sinks", PARTS)
def test_window_in_parts(eng, b, lq, lk, h, hk, d, dtype, buckets, causal, before, after, sinks):
    say("window in parts", b, lq, lk, h, hk, d, dtype, buckets, causal, before, after, sinks)
    tensors, doubles, lengths = attention_inputs(b, lq, lk, h, hk, d, dtype, buckets, False, seed=131)
    hold(tensors, doubles, 1 / math.sqrt(d), dtype, before, after, sinks, lengths, causal=causal, max_distance=128)


# A value rounded once is off by at most U relative to it, evenly: a tensor so rounded by at most U / sqrt(3) of its norm.
# Where the products take p and ds in 16 bits, those roundings are as large and independent: sqrt(2) times that.  The
# second sum of squares is of few values, or falls on few p: 5 standard deviations of a mean of 1000 evenly spread
# squares (sqrt(0.8 / 1000) each) give 1.07, and fp32 sums add less than a thousandth.
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("b,lq,lk,h,hk,d,buckets,causal,before,after,sinks", [
    (8, 1, 700, 2, 2, 64, 0, False, 20, 200, 0), (16, 1, 500, 2, 1, 64, 32, True, 245, 0, 4), (4, 3, 300, 4, 4, 128, 0, True, 260, 0, 0),
    (3, 600, 900, 16, 8, 32, 64, True, 166, 0, 0), (2, 500, 500, 16, 16, 64, 32, False, 90, 90, 1), (1, 700, 700, 4, 2, 128, 0, True, 300, 0, 4)])
def test_window_errors_are_the_roundings(eng, dtype, b, lq, lk, h, hk, d, buckets, causal, before, after, sinks):
    say("window errors", dtype, b, lq, lk, h, hk, d, buckets, causal, before, after, sinks)
    (q, k, v, do, table), (qd, kd, vd, dod, td), _ = attention_inputs(b, lq, lk, h, hk, d, dtype, buckets, False, seed=136)
    args = dict(causal=causal, max_distance=128)
    want = lo.window_attention(qd, kd, vd, dod, d**-0.5, dtype, before, after, sinks, td, **args)
    out, lse = encoder.attention_forward(q, k, v, table, window=(before, after), sinks=sinks, scale=d**-0.5, **args)
    got = encoder.attention_backward(do, q, k, v, out, lse, table, window=(before, after), sinks=sinks, scale=d**-0.5, **args)
    few = lq * (h // hk) < 128
    for name, a in zip(("out", *GRADS), (out, *got)):
        if a is None:
            continue
        exact = want[name][0].double()
        roundings = 1 if few or name in ("dq", "dtable") else 2
        off = float((a.double().cpu() - exact).norm() / exact.norm())
        assert off <= 1.07 * o.U[dtype] * math.sqrt(roundings / 3), (name, off / o.U[dtype])


@pytest.mark.parametrize("lq,start", [(1, [0, 57, 199]), (4, [3, 100, 150]), (70, [-80, 0, 129]), (40, [-20, -39, 500]), (200, [-100, 150, 0])])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("before,after,sinks", [(30, 5, 0), (2, 80, 3), (0, 0, 0), (150, 0, 40)])
def test_window_query_start(eng, lq, start, causal, before, after, sinks):
    """Rows at positions of their own, some before the first key or past the last one, in caches of ragged length."""
    tensors, doubles, _ = attention_inputs(3, lq, 200, 4, 2, 64, BF16, 0, False, seed=141)
    lengths = {"key_lengths": torch.tensor([200, 60, 199], dtype=torch.int32), "query_start": torch.tensor(start, dtype=torch.int32)}
    hold(tensors, doubles, 0.2, BF16, before, after, sinks, lengths, causal=causal)


def test_window_lengths_of_zero_and_short(eng):
    for dtype in (F16, BF16):
        tensors, doubles, _ = attention_inputs(5, 150, 150, 2, 2, 32, dtype, 8, False, seed=151)
        lengths = {"key_lengths": torch.tensor([0, 1, 63, 64, 150], dtype=torch.int32),
                   "query_lengths": torch.tensor([150, 150, 0, 1, 130], dtype=torch.int32)}
        for causal in (False, True):
            for before, after, sinks in ((10, 10, 0), (70, 30, 2), (0, 0, 150)):
                hold(tensors, doubles, 0.2, dtype, before, after, sinks, lengths, causal=causal, max_distance=20)


def test_window_that_hides_nothing_is_attention(eng):
    """Windows and first keys as long as the sequence, or longer than any."""
    tensors, doubles, _ = attention_inputs(2, 300, 300, 4, 2, 64, BF16, 32, False, seed=161)
    for causal in (False, True):
        for before, after, sinks in ((299, 299, 0), (1 << 40, 1 << 40, 0), (1 << 62, 0 if causal else 1 << 33, 1 << 50), (0, 0, 300)):
            hold(tensors, doubles, 0.125, BF16, before, after, sinks, {}, causal=causal, max_distance=100)


def test_window_of_one_key_has_no_score_gradient(eng):
    """Where every row sees one key, ds is zero, and so are dq and dk, exactly; dv is dout."""
    for dtype in (F16, BF16):
        for d in (32, 64, 128):
            (q, k, v, do, _), (_, _, _, dod, _), _ = attention_inputs(2, 200, 200, 2, 2, d, dtype, 0, False, seed=171)
            for causal in (False, True):
                out, lse = encoder.attention_forward(q, k, v, window=0, causal=causal)
                assert torch.equal(out, v)
                dq, dk, dv, _ = encoder.attention_backward(do, q, k, v, out, lse, window=0, causal=causal)
                assert not dq.any() and not dk.any() and torch.equal(dv, do)
            out, lse = encoder.attention_forward(q, k, v, window=(0, 0), sinks=1, query_start=torch.full((2,), 300, dtype=torch.int32, device="cuda"))
            assert torch.equal(out, v[:, :1].expand_as(out))
            dq, dk, dv, _ = encoder.attention_backward(do, q, k, v, out, lse, window=0, sinks=1,
                                                       query_start=torch.full((2,), 300, dtype=torch.int32, device="cuda"))
            assert not dq.any() and not dk.any() and not dv[:, 1:].any()
            want = dod.sum(1, keepdim=True)
            o.within(dv[:, :1], want, o.U[dtype] * want.abs() + 200 * o.F32 * dod.abs().sum(1, keepdim=True), "dv of the first key")


def test_window_large_cache_of_single_tokens(eng):
    """The window's keys, and the first ones, are all that is read: the rest of the cache may hold anything."""
    g = torch.Generator().manual_seed(9)
    b, lk, h, hk, d = 3, 5000, 8, 2, 128
    q = torch.randn(b, 1, h, d, generator=g).to(F16)
    k, v = (torch.randn(b, lk, hk, d, generator=g).to(F16) for _ in range(2))
    kl = torch.tensor([5000, 1203, 4], dtype=torch.int32)
    start = kl - 1
    kk, vv = k.clone(), v.clone()
    for n in range(b):
        for t in (kk, vv):
            t[n, 4:max(4, int(start[n]) - 1024)] = math.nan
            t[n, int(kl[n]):] = math.inf
    args = dict(window=(1024, 0), sinks=4, causal=True, key_lengths=kl.cuda(), query_start=start.cuda())
    out, lse = encoder.attention_forward(q.cuda(), kk.cuda(), vv.cuda(), **args)
    want = lo.window_attention(q.double(), k.double(), v.double(), q.double(), d**-0.5, F16, 1024, 0, 4, causal=True, key_lengths=kl, query_start=start)
    o.within(out, *want["out"], "out")
    o.within(lse, *want["lse"], "lse")


def test_window_strides_and_offsets(eng):
    """Views of one projection's output, other orders of the dimensions, expanded heads, odd offsets."""
    b, l, h, d = 2, 170, 4, 32
    qkv = torch.randn(b, l, 3, h, d, device="cuda").to(F16)
    odd = torch.randn(b * l * h * d + 1, device="cuda").to(F16)[1:].view(b, l, h, d)
    other = torch.randn(h, b, l, d, device="cuda").to(F16).permute(1, 2, 0, 3)
    one = torch.randn(b, l, 1, d, device="cuda").to(F16).expand(b, l, h, d)
    more = dict(window=(40, 25), sinks=3)
    for q, k, v in ((qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]), (odd, other, one)):
        out, lse = encoder.attention_forward(q, k, v, **more)
        want, lsec = encoder.attention_forward(q.contiguous(), k.contiguous(), v.contiguous(), **more)
        assert torch.equal(out, want) and torch.equal(lse, lsec)
        for do in (odd, other, one):
            a = encoder.attention_backward(do, q, k, v, out, lse, **more)
            w = encoder.attention_backward(do.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), out, lse, **more)
            assert all(torch.equal(x, y) for x, y in zip(a[:3], w[:3]))


def test_window_empty(eng):
    def t(*shape):
        return torch.randn(*shape, device="cuda").to(F16)

    q, k = t(2, 5, 2, 16), t(2, 0, 2, 16)
    out, lse = encoder.attention_forward(q, k, k, window=3, sinks=2)
    assert not out.any() and torch.isinf(lse).all()
    assert not encoder.attention_backward(q, q, k, k, out, lse, window=3, sinks=2)[0].any()
    out, lse = encoder.attention_forward(k, q, q, window=3, sinks=2)
    assert out.shape == k.shape
    _, dk, dv, _ = encoder.attention_backward(k, k, q, q, out, lse, window=3, sinks=2)
    assert not dk.any() and not dv.any()


def test_window_small_and_large_gradients_of_float16(eng):
    """Gradients at both ends of float16's range keep their digits, the first keys' too."""
    l, d = 2000, 32
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(1, l, 1, d, generator=g).to(F16) * s for s in (0.1, 0.1, 1.0))
    more = dict(window=(900, 300), sinks=5)
    out, lse = encoder.attention_forward(q.cuda(), k.cuda(), v.cuda(), **more)
    for size in (2.0**-12, 1.0, 2.0**9):
        do = (torch.randn(1, l, 1, d, generator=g) * size).to(F16)
        grads = encoder.attention_backward(do.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse, **more)
        want = lo.window_attention(q.double(), k.double(), v.double(), do.double(), d**-0.5, F16, 900, 300, 5)
        for name, a in zip(GRADS[:3], grads):
            for part in (slice(0, 5), slice(5, None)):
                r, x = want[name][0][:, part], a.double().cpu()[:, part]
                rel = float((x - r).norm() / r.norm())
                # half the spacing of the result's subnormals, relative to its size, and a few roundings of operands
                room = 2.0**-25 / float(r.square().mean().sqrt()) + 4 * 2.0**-11
                assert rel <= room, f"{name} at {size}: {rel} of {room}"


def test_window_through_autograd_and_against_differences(eng):
    """A layer with windowed attention and the gated block: the gradients' product with a direction is the
    change of the 64-bit forward along it."""
    torch.manual_seed(7)
    b, l, h, d, f = 2, 90, 2, 16, 32
    t = {n: (torch.randn(*s) * c).to(BF16) for n, s, c in (
        ("x", (b, l, f), 1.0), ("w", (3 * f, f), 0.3), ("table", (8, h), 1.0), ("gate", (48, f), 0.25), ("up", (48, f), 0.25),
        ("down", (f, 48), 0.2), ("g", (f,), 1.0))}
    weight = torch.randn(b, l, f).to(BF16)

    def ours(p):
        qkv = encoder.linear(p["x"], p["w"]).view(b, l, 3, h, d)
        a = encoder.attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], p["table"], max_distance=20, window=(12, 7), sinks=2)
        y = encoder.linear(encoder.gated_linear(a.view(b, l, f), p["gate"], p["up"]), p["down"], residual=p["x"])
        return encoder.layer_norm(y, p["g"])

    def plain(p):
        qkv = (p["x"] @ p["w"].T).view(b, l, 3, h, d)
        a = lo.window_attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], qkv[:, :, 0], 0.25, BF16, 12, 7, 2, p["table"], 20)["out"][0]
        y = lo.gated(a.reshape(b, l, f), p["gate"], p["up"], None, None, "silu")[0] @ p["down"].T + p["x"]
        return o.norm(y, p["g"], None, 1e-5)[0]

    dev = {n: v.cuda().requires_grad_() for n, v in t.items()}
    (ours(dev) * weight.cuda()).float().sum().backward()
    base = {n: v.double() for n, v in t.items()}
    for n in t:
        step = torch.randn(t[n].shape, dtype=torch.float64)
        eps = 1e-5
        change = [(plain({**base, n: base[n] + s * eps * step}) * weight.double()).sum() for s in (1, -1)]
        want = float(change[0] - change[1]) / (2 * eps)
        got = float((dev[n].grad.double().cpu() * step).sum())
        room = 10 * o.U[BF16] * float(dev[n].grad.double().norm())  # each of the chain's roundings gives a few U of the gradient's norm
        assert abs(got - want) <= room, f"{n}: {got}, {want} by differences, {room}"


def test_window_of_a_call_counts(eng):
    """Calls that differ in their window only, by number, pair, tensor: each by its own."""
    (q, k, v, do, _), doubles, _ = attention_inputs(1, 200, 200, 2, 2, 32, F16, 0, False, seed=181)
    qd, kd, vd, dod, _ = doubles
    for window, sinks, before, after in ((9, 0, 9, 9), ((3, 50), 2, 3, 50), (torch.tensor(9), 1, 9, 9), ([70, 0], 0, 70, 0)):
        want = lo.window_attention(qd, kd, vd, dod, 32**-0.5, F16, before, after, sinks)
        out, lse = encoder.attention_forward(q, k, v, window=window, sinks=sinks)
        o.within(out, *want["out"], "out")
        dq = encoder.attention_backward(do, q, k, v, out, lse, window=window, sinks=sinks)[0]
        o.within(dq, *want["dq"], "dq")
    pair = [5, 5]
    qq = q.clone().requires_grad_()
    y = encoder.attention(qq, k, v, window=pair, sinks=1)
    pair[0] = 100  # (the forward pass's window is the backward pass's)
    y.backward(do)
    o.within(qq.grad, *lo.window_attention(qd, kd, vd, dod, 32**-0.5, F16, 5, 5, 1)["dq"], "dq")


def test_window_refusals(eng):
    def t(*shape):
        return torch.randn(*shape, device="cuda").to(F16)

    q = t(1, 20, 2, 16)
    for more, reason in (({"sinks": 3}, "need a window"), ({"window": -1}, "negative"), ({"window": (3, -2)}, "negative"),
                         ({"window": 3, "sinks": -1}, "negative")):
        with pytest.raises(RuntimeError, match=reason):
            encoder.attention(q, q, q, **more)
    for more in ({"window": 2.5}, {"window": (1, 2, 3)}, {"window": 4, "sinks": 1.5}, {"window": "12"}):
        with pytest.raises((TypeError, ValueError)):
            encoder.attention(q, q, q, **more)


def test_layer_on_other_streams_and_graph_replays(eng):
    """The operators of a layer, on a stream of the caller's own and captured: every replay gives the eager result."""
    torch.manual_seed(10)
    x = torch.randn(3, 150, 64, device="cuda").to(F16)
    w = (torch.randn(192, 64, device="cuda") * 0.2).to(F16)
    gate, up, down = ((torch.randn(*s, device="cuda") * 0.2).to(F16) for s in ((96, 64), (96, 64), (64, 96)))
    table = torch.randn(8, 4, device="cuda").to(F16)
    values, scales = encoder.quantize_rows(down)
    more = dict(max_distance=30, window=(40, 20), sinks=3)

    def step():
        qkv, _ = encoder.linear_forward(x, w)
        q, k, v = qkv.view(3, 150, 3, 4, 16).unbind(2)
        out, lse = encoder.attention_forward(q, k, v, table, **more)
        a = out.view(3, 150, 64)
        hidden, pre = encoder.gated_linear_forward(a, gate, up, keep_pre=True)
        y = encoder.linear_int8(hidden, values, scales, residual=x)
        token = encoder.linear_int8(hidden[:1, :1], values, scales)
        one = encoder.attention_forward(q[:, -1:], k, v, causal=True, window=(30, 0), sinks=2)[0]
        grads = encoder.gated_linear_backward(hidden, a, gate, up, pre)
        return (y, token, one, *grads, *encoder.attention_backward(grads[0].view_as(q), q, k, v, out, lse, table, **more))

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


def test_few_rows_on_two_streams_and_in_graphs(eng):
    """Calls of few rows, narrow windows and split key axes, at once on two streams and as two graphs whose replays alternate:
    each has its own scratch, and changed inputs are read anew."""
    torch.manual_seed(11)

    def make(lq, h, d, dtype, buckets, before, sinks):
        q, do = (torch.randn(2, lq, h, d, device="cuda").to(dtype) for _ in range(2))
        k, v = (torch.randn(2, 1300, h, d, device="cuda").to(dtype) for _ in range(2))
        table = torch.randn(buckets, h, device="cuda").to(dtype) if buckets else None
        x, dy = torch.randn(lq, 64, device="cuda").to(dtype), torch.randn(lq, 40, device="cuda").to(dtype)
        gate, up = (torch.randn(40, 64, device="cuda").to(dtype) for _ in range(2))
        more = dict(causal=True, window=(before, 0), sinks=sinks, max_distance=100)

        def step():
            out, lse = encoder.attention_forward(q, k, v, table, **more)
            grads = encoder.attention_backward(do, q, k, v, out, lse, table, **more)
            _, pre = encoder.gated_linear_forward(x, gate, up, keep_pre=True)
            return [t for t in (out, lse, *grads, *encoder.gated_linear_backward(dy, x, gate, up, pre)) if t is not None]

        return step, (q, do, x, dy)

    forms = [(1, 4, 64, BF16, 32, 900, 0), (5, 2, 128, F16, 0, 30, 2), (32, 1, 32, BF16, 16, 1200, 4), (130, 1, 64, F16, 0, 1299, 0)]
    made = [make(*form) for form in forms]
    want = [[t.clone() for t in step()] for step, _ in made]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        got = []
        for n, (step, _) in enumerate(made):
            with torch.cuda.stream(sides[n % 2]):
                got.append(step())
        for side in sides:
            side.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, held = [], []
    for step, _ in made:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step())
    for turn in range(3):
        for _, inputs in made:
            for t in inputs:
                t.mul_(0.75)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (step, _), results in zip(made, held):
            assert all(torch.equal(a, b) for a, b in zip(results, step()))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("b,lq,lk,h,d,buckets,causal,before,after,sinks", [
    (2, 200, 200, 2, 64, 32, False, 40, 40, 1), (1, 300, 300, 1, 128, 16, True, 200, 0, 0), (2, 3, 150, 2, 32, 8, False, 3, 3, 0),
    (1, 130, 130, 2, 64, 32, False, 10, 10, 0)])
def test_window_with_infinite_bias(eng, dtype, b, lq, lk, h, d, buckets, causal, before, after, sinks):
    """Buckets of minus infinity hide keys as the mask does: some of a row's, or all."""
    tensors, doubles, _ = attention_inputs(b, lq, lk, h, h, d, dtype, buckets, False, seed=77)
    for hidden in ([0], [1, 2, 3], list(range(buckets // 2)), list(range(buckets))):
        say("infinite bias", dtype, b, lq, lk, h, d, buckets, causal, before, after, sinks, hidden)
        table, exact = tensors[4].clone(), doubles[4].clone()
        table[hidden, 0] = exact[hidden, 0] = -math.inf
        hold((*tensors[:4], table), (*doubles[:4], exact), 1 / math.sqrt(d), dtype, before, after, sinks, {}, causal=causal,
             max_distance=128, poison=False)
