"""What lies in places that no row sees, or in rows that see nothing, reaches no result of
attention: NaN and infinities there (memory that nobody wrote) change nothing (needs an MI355X).
"""

from __future__ import annotations

import math

import pytest
import torch

import encoder_oracle as o
from cuda_vector_search import encoder

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def make(b, lq, lk, h, hk, d, dtype, buckets, seed=61):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype)

    return rand(b, lq, h, d, scale=1.5), rand(b, lk, hk, d), rand(b, lk, hk, d), rand(b, lq, h, d, scale=0.5), \
        rand(buckets, h) if buckets else None


# batch, lq, lk, heads, key heads, width, type, buckets, start, key lengths: causal
CACHES = [
    (2, 1, 200, 4, 2, 64, F16, 0, [57, 130], None),       # single tokens over a cache filled so far
    (2, 1, 200, 4, 4, 64, BF16, 32, [0, 199], None),
    (2, 1, 3000, 4, 1, 128, F16, 0, [1029, 2100], None),  # in parts
    (2, 4, 333, 8, 2, 40, BF16, 0, [5, 100], [400, 90]),
    (2, 70, 300, 2, 2, 64, F16, 32, [3, 200], None),      # more rows than one block's columns
    (1, 130, 2500, 2, 1, 128, BF16, 0, [777], None),
    (2, 70, 200, 2, 2, 64, BF16, 16, [-20, 40], None),    # rows that see nothing
    (1, 129, 31, 2, 1, 72, F16, 0, [-98], None),
    (2, 40, 500, 2, 2, 32, F16, 0, [-39, -60], None),
]


@pytest.mark.parametrize("filler", [math.nan, math.inf])
@pytest.mark.parametrize("b,lq,lk,h,hk,d,dtype,buckets,start,lengths", CACHES)
def test_causal_cache_with_unwritten_places(eng, b, lq, lk, h, hk, d, dtype, buckets, start, lengths, filler):
    print("cache", b, lq, lk, h, hk, d, dtype, buckets, start, filler, flush=True)
    q, k, v, do, table = make(b, lq, lk, h, hk, d, dtype, buckets)
    ref = dict(causal=True, query_start=torch.tensor(start, dtype=torch.int32), max_distance=100)
    if lengths is not None:
        ref["key_lengths"] = torch.tensor(lengths, dtype=torch.int32)
    exact = [t.double() for t in (q, k, v, do)]
    for n, at in enumerate(start):
        k[n, max(at + lq, 0):] = filler
        v[n, max(at + lq, 0):] = filler
        q[n, :max(-at, 0)] = filler
        do[n, :max(-at, 0)] = filler
    more = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in ref.items()}
    q, k, v, do = (t.cuda() for t in (q, k, v, do))
    table_gpu = None if table is None else table.cuda()
    ref["table"] = None if table is None else table.double()
    qd, kd, vd, dod = exact
    out, lse = encoder.attention_forward(q, k, v, table_gpu, scale=0.2, **more)
    want, bound = o.attention(qd, kd, vd, 0.2, **ref), o.attention_bounds(qd, kd, vd, 0.2, dtype, **ref)
    o.within(out, want[0], bound[0], "out")
    o.within(lse, want[1], bound[1], "lse")
    grads = encoder.attention_backward(do, q, k, v, out, lse, table_gpu, scale=0.2, **more)
    for name, a, r, t in zip(("dq", "dk", "dv", "dtable"), grads, o.attention_grads(dod, qd, kd, vd, 0.2, **ref),
                             o.attention_grad_bounds(dod, qd, kd, vd, 0.2, dtype, **ref)):
        if r is not None:
            o.within(a, r, t, name)


@pytest.mark.parametrize("lq,lk,h,hk,d,buckets", [(20, 30, 2, 2, 64, 8), (20, 3000, 2, 2, 32, 0), (300, 300, 2, 1, 64, 0),
                                                   (200, 4000, 1, 1, 128, 32)])
def test_rows_past_the_end_are_zero_beside_infinite_values(eng, lq, lk, h, hk, d, buckets):
    """A value that is not finite reaches the rows that see it, and no row past the sequence's end."""
    print("padded rows", lq, lk, h, hk, d, buckets, flush=True)
    q, k, v, do, table = make(2, lq, lk, h, hk, d, F16, buckets)
    v[0, 3], v[1, lk - 1] = math.nan, math.inf
    q, k, v, do = (t.cuda() for t in (q, k, v, do))
    table = None if table is None else table.cuda()
    ql = torch.tensor([lq // 2, lq - 3], dtype=torch.int32, device="cuda")
    more = dict(query_lengths=ql, max_distance=100)
    out, lse = encoder.attention_forward(q, k, v, table, **more)
    dq = encoder.attention_backward(do, q, k, v, out, lse, table, **more)[0]
    for n in range(2):
        at = int(ql[n])
        assert not out[n, at:].any() and (lse[n, :, at:] == -math.inf).all() and not dq[n, at:].any()
        assert not torch.isfinite(out[n, :at]).any()
