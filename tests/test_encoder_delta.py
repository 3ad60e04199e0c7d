"""Attention's gradient in rows that see few keys: their ds is small beside its terms, so dout . out has
to come from the probabilities, not from ``out`` in 16 bits (needs an MI355X).
"""

from __future__ import annotations

import math

import pytest
import torch

import encoder_oracle as o
from cuda_vector_search import encoder
from encoder_tight import grad_bounds

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def tile(d):
    """Keys of a tile of the kernel that sums over keys."""
    return 32 if d > 64 else 64


# batch, lq, lk, heads, key heads, width, type, buckets, query start or None, ragged
CASES = [
    (1, 65, 65, 2, 2, 64, BF16, 0, None, False), (1, 65, 65, 2, 2, 64, F16, 0, None, False),
    (2, 300, 300, 2, 1, 64, BF16, 32, None, True), (1, 100, 100, 2, 2, 128, BF16, 0, None, False),
    (1, 200, 200, 4, 2, 32, F16, 16, None, False), (2, 90, 400, 2, 2, 64, BF16, 0, [-10, 13], False),
    (1, 1100, 1100, 2, 1, 64, BF16, 0, None, False),  # the keys in parts
    (2, 160, 1600, 3, 1, 128, F16, 0, [0, -45], False),
]


@pytest.mark.parametrize("b,lq,lk,h,hk,d,dtype,buckets,start,ragged", CASES)
def test_first_causal_rows(eng, b, lq, lk, h, hk, d, dtype, buckets, start, ragged):
    print("first rows", b, lq, lk, h, hk, d, dtype, buckets, start, ragged, flush=True)
    g = torch.Generator().manual_seed(71)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype)

    q, k, v, do = rand(b, lq, h, d, scale=3.0), rand(b, lk, hk, d), rand(b, lk, hk, d), rand(b, lq, h, d)
    table = rand(buckets, h) if buckets else None
    scale = 1 / math.sqrt(d)
    ref = dict(causal=True, max_distance=100)
    if start is not None:
        ref["query_start"] = torch.tensor(start, dtype=torch.int32)
    if ragged:
        ref["key_lengths"] = ref["query_lengths"] = torch.tensor([lk - 70 * n for n in range(b)], dtype=torch.int32)
    more = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in ref.items()}
    args = [t.cuda() for t in (q, k, v)]
    table_gpu = None if table is None else table.cuda()
    out, lse = encoder.attention_forward(*args, table_gpu, **more)
    got = encoder.attention_backward(do.cuda(), *args, out, lse, table_gpu, **more)
    # blocks of 32 rows whose last one sees at most one tile, in every sequence
    last_start = lk - lq if start is None else max(start)
    own = (torch.arange(lq) // 32 + 1) * 32 + last_start <= tile(d)
    assert own.any() or d > 64
    ref["table"] = None if table is None else table.double()
    want, bounds = grad_bounds(do.double(), q.double(), k.double(), v.double(), scale, dtype, own_delta=own, **ref)
    for name, a, r, t in zip(("dq", "dk", "dv", "dtable"), got, want, bounds):
        if r is not None:
            o.within(a, r, t, name)
