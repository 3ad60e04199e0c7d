"""The encoder operators where a long axis is cut into parts that are joined (needs an MI355X).

Each case asserts, by the workspace its plan asks for, that the parts it is about are in use.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import encoder_oracle as o
from cuda_vector_search import _ext, encoder

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def up256(n):
    return (n + 255) // 256 * 256


def attention_bytes(q, k, buckets, causal, backward):
    b, lq, h, d = q.shape
    a = _ext.AttentionArgs(batch=b, q_len=lq, k_len=k.shape[1], heads=h, k_heads=k.shape[2], width=d, scale=1.0,
                           type=encoder.TYPES[q.dtype], causal=causal, buckets=buckets, max_distance=128)
    if buckets:
        a.bias_table = q.data_ptr()
    out = ctypes.c_int64()
    assert _ext.load().lib.cvs_attention_plan(ctypes.byref(a), backward, q.device.index, ctypes.byref(out)) == 0
    return out.value


def backward_parts(q, k, buckets, causal):
    """(parts of the keys for dq, parts of the queries for dk and dv) that the plan's bytes stand for,
    of at least 512 keys and 8 tiles of 64 queries each."""
    b, lq, h, d = q.shape
    rows, blocks = b * h * lq, (lq + 127) // 128
    size = attention_bytes(q, k, buckets, causal, 1)
    found = []
    for qp in range(1, max(1, k.shape[1] // 512) + 1):
        for kp in range(1, max(1, (lq + 63) // 64 * (h // k.shape[2]) // 8) + 1):
            need = up256(rows * 4) + (up256(qp * rows * d * 4) if qp > 1 else 0)
            need += up256(b * h * qp * blocks * 4) if q.dtype == F16 else 0
            need += up256(h * b * qp * blocks * buckets * 4) if buckets else 0
            need += up256(kp * 2 * k.numel() * 4) if kp > 1 else 0
            if need == size:
                found.append((qp, kp))
    assert len(found) == 1, f"{size} bytes: {found}"
    return found[0]


def inputs(b, lq, lk, h, hk, d, dtype, buckets, seed=101):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype)

    return (rand(b, lq, h, d, scale=1.5), rand(b, lk, hk, d), rand(b, lk, hk, d), rand(b, lq, h, d, scale=0.5),
            rand(buckets, h) if buckets else None)


# batch, lq, lk, heads, key heads, width, type, buckets, causal, lengths, which parts are several (dq's, dk's)
BACKWARD = [
    (1, 1100, 1100, 4, 2, 128, BF16, 0, True, None, (True, True)),
    (2, 1100, 1100, 2, 1, 64, BF16, 32, False, [1100, 20], (True, True)),   # a sequence of one tile beside a long one
    (2, 1100, 1100, 2, 1, 64, F16, 32, True, [1030, 64], (True, True)),
    (1, 777, 1029, 6, 2, 64, F16, 0, True, None, (True, True)),             # parts that end inside a head's queries
    (1, 1000, 300, 3, 1, 72, F16, 16, True, [290], (False, True)),
    (3, 600, 90, 3, 1, 32, BF16, 0, False, [90, 1, 0], (False, True)),
    (1, 100, 1600, 3, 3, 40, BF16, 8, True, [1500], (True, False)),
    (2, 1, 2048, 4, 2, 128, F16, 0, False, [2048, 33], (True, False)),
]


@pytest.mark.parametrize("b,lq,lk,h,hk,d,dtype,buckets,causal,lengths,several", BACKWARD)
def test_attention_backward_parts(eng, b, lq, lk, h, hk, d, dtype, buckets, causal, lengths, several):
    print("backward parts", b, lq, lk, h, hk, d, dtype, buckets, causal, lengths, flush=True)
    q, k, v, do, table = inputs(b, lq, lk, h, hk, d, dtype, buckets)
    ref = dict(causal=causal, max_distance=128)
    if lengths is not None:
        ref["key_lengths"] = torch.tensor(lengths, dtype=torch.int32)
        if lq == lk:
            ref["query_lengths"] = ref["key_lengths"]
    more = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in ref.items()}
    args = [t.cuda() for t in (q, k, v)]
    table_gpu = None if table is None else table.cuda()
    parts = backward_parts(args[0], args[1], buckets, causal)
    assert (parts[0] > 1, parts[1] > 1) == several, f"parts {parts}"
    out, lse = encoder.attention_forward(*args, table_gpu, **more)
    got = encoder.attention_backward(do.cuda(), *args, out, lse, table_gpu, **more)
    again = encoder.attention_backward(do.cuda(), *args, out, lse, table_gpu, **more)
    assert all(x is None or torch.equal(x, y) for x, y in zip(got, again))
    exact = [t.double() for t in (q, k, v)]
    ref["table"] = None if table is None else table.double()
    scale = 1 / math.sqrt(d)
    for name, a, r, t in zip(("dq", "dk", "dv", "dtable"), got, o.attention_grads(do.double(), *exact, scale, **ref),
                             o.attention_grad_bounds(do.double(), *exact, scale, dtype, **ref)):
        if r is not None:
            o.within(a, r, t, name)


# batch, lq, lk, heads, key heads, width, type, buckets, causal, key lengths
FORWARD = [
    (1, 5, 2048, 4, 1, 64, F16, 0, False, None),     # shared heads' rows in one block
    (2, 2, 3000, 24, 2, 128, BF16, 0, True, [3000, 700]),
    (1, 1, 5000, 8, 8, 40, F16, 0, False, [4999]),
    (1, 3, 2100, 4, 2, 32, BF16, 32, False, None),   # a bias: a head a block
    (1, 100, 2000, 3, 1, 64, F16, 0, True, None),    # blocks of 128 rows
    (2, 70, 1500, 2, 2, 128, BF16, 16, False, [1500, 100]),
]


@pytest.mark.parametrize("b,lq,lk,h,hk,d,dtype,buckets,causal,lengths", FORWARD)
def test_attention_forward_parts(eng, b, lq, lk, h, hk, d, dtype, buckets, causal, lengths):
    print("forward parts", b, lq, lk, h, hk, d, dtype, buckets, causal, lengths, flush=True)
    q, k, v, _, table = inputs(b, lq, lk, h, hk, d, dtype, buckets)
    ref = dict(causal=causal, max_distance=128)
    if lengths is not None:
        ref["key_lengths"] = torch.tensor(lengths, dtype=torch.int32)
    more = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in ref.items()}
    args = [t.cuda() for t in (q, k, v)]
    assert attention_bytes(args[0], args[1], buckets, causal, 0) > 0, "in one part"
    out, lse = encoder.attention_forward(*args, None if table is None else table.cuda(), **more)
    ref["table"] = None if table is None else table.double()
    exact = [t.double() for t in (q, k, v)]
    scale = 1 / math.sqrt(d)
    for name, a, r, t in zip(("out", "lse"), (out, lse), o.attention(*exact, scale, **ref), o.attention_bounds(*exact, scale, dtype, **ref)):
        o.within(a, r, t, name)


@pytest.mark.parametrize("lq,lk,h,hk", [(3, 50, 2, 2), (4, 2100, 4, 1), (200, 200, 2, 1), (100, 1500, 2, 2)])
def test_attention_values_that_are_not_finite(eng, lq, lk, h, hk):
    """A NaN in q is its row's, one in k or v every row's that sees it."""
    q, k, v, _, _ = inputs(1, lq, lk, h, hk, 64, F16, 0)
    plain = encoder.attention(q.cuda(), k.cuda(), v.cuda())
    spoilt = q.clone()
    spoilt[0, 1, 0, 3] = math.nan
    out, lse = encoder.attention_forward(spoilt.cuda(), k.cuda(), v.cuda())
    assert torch.isnan(out[0, 1, 0]).all() and torch.isnan(lse[0, 0, 1])
    keep = torch.ones(lq, h, dtype=torch.bool, device="cuda")
    keep[1, 0] = False
    assert torch.equal(out[0][keep], plain[0][keep])
    for value in (math.nan, math.inf, -math.inf):
        at = lk - 7
        kk, vv = k.clone(), v.clone()
        kk[0, at, 0, 5], vv[0, at, 0, 5] = value, value
        shares = slice(0, h // hk)  # the query heads of key head 0
        out = encoder.attention(q.cuda(), kk.cuda(), v.cuda())
        if math.isnan(value):
            assert torch.isnan(out[0, :, shares]).all()
        assert torch.equal(out[0, :, h // hk:], plain[0, :, h // hk:])
        out = encoder.attention(q.cuda(), k.cuda(), vv.cuda())
        assert not torch.isfinite(out[0, :, shares, 5]).any()
        other = [c for c in range(64) if c != 5]
        assert torch.equal(out[0, :, :, other], plain[0, :, :, other])


@pytest.mark.parametrize("rows,width,dtype", [(40001, 24, F16), (33000, 133, F32), (70000, 72, BF16)])
def test_layer_norm_gradients_of_many_rows(eng, rows, width, dtype):
    """More than 128 rows a CU: fewer workgroups, each with more of them."""
    g = torch.Generator().manual_seed(111)
    x, dy = ((torch.randn(rows, width, generator=g) + c).to(dtype) for c in (0.3, 0.0))
    w = (1 + 0.2 * torch.randn(width, generator=g)).to(dtype)
    y, mean, rstd = encoder.layer_norm_forward(x.cuda(), w.cuda())
    got = encoder.layer_norm_backward(dy.cuda(), x.cuda(), w.cuda(), mean, rstd)
    args = dy.double(), x.double(), w.double(), mean.double().cpu(), rstd.double().cpu()
    for name, a, r, t in zip(("dx", "dweight", "dbias"), got, o.norm_grads(*args), o.norm_grad_bounds(*args, dtype)):
        o.within(a, r, t, name)


def test_layer_norm_of_more_rows_than_a_launch(eng):
    """2^23 rows and some: launches of pieces, the same bits as pieces of the caller's."""
    rows, at = 2**23 + 5, 2**23 - 50
    x = torch.randn(rows, 8, device="cuda", dtype=F16)
    w, b = torch.randn(8, device="cuda").to(F16), torch.randn(8, device="cuda").to(F16)
    y, mean, rstd = encoder.layer_norm_forward(x, w, b)
    for part in (slice(0, 100), slice(at, rows)):
        for a, r in zip((y[part], mean[part], rstd[part]), encoder.layer_norm_forward(x[part].contiguous(), w, b)):
            assert torch.equal(a, r)
