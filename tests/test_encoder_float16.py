"""Attention's gradients in float16 keep their digits where the products' operands, ds and the
probabilities, would be subnormal or infinite as float16 numbers (needs an MI355X).
"""

from __future__ import annotations

import math

import pytest
import torch

import encoder_oracle as o
from cuda_vector_search import encoder
from encoder_tight import grad_bounds

pytestmark = pytest.mark.gpu

F16 = torch.float16
LIFT = 14  # (tighter than the 2^10 the kernels lift by: these inputs leave that room)


def gradients(q, k, v, do, table=None, scale=None, **more):
    more = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in more.items()}
    q, k, v, do = (t.cuda() for t in (q, k, v, do))
    table = None if table is None else table.cuda()
    out, lse = encoder.attention_forward(q, k, v, table, scale=scale, **more)
    return encoder.attention_backward(do, q, k, v, out, lse, table, scale=scale, **more)


@pytest.mark.parametrize("size", [2.0**-12, 1.0, 2.0**9])
@pytest.mark.parametrize("lq,lk,d", [(3000, 3000, 32), (512, 8192, 64), (8192, 512, 64), (1500, 1500, 128)])
def test_long_rows(eng, lq, lk, d, size):
    """Rows of many keys, gradients at both ends of float16's range."""
    print("long rows", lq, lk, d, size, flush=True)
    g = torch.Generator().manual_seed(81)
    q, k, v = (torch.randn(1, l, 1, d, generator=g).to(F16) for l in (lq, lk, lk))
    do = (torch.randn(1, lq, 1, d, generator=g) * size).to(F16)
    want = o.attention_grads(do.double(), q.double(), k.double(), v.double(), 1 / math.sqrt(d))
    for name, a, r in zip(("dq", "dk", "dv"), gradients(q, k, v, do), want):
        rel = float((a.double().cpu() - r).norm() / r.norm())
        # half the spacing of the result's subnormals, relative to its size, and a few roundings of operands
        room = 2.0**-25 / float(r.square().mean().sqrt()) + 4 * 2.0**-11
        assert rel <= room, f"{name}: {rel} of {room}"


# lq, lk, heads, key heads, width, buckets, causal, sharpness of the softmax, sizes of dout (powers of two)
CASES = [
    (200, 900, 2, 2, 64, 0, False, 1.0, (-13, 10)), (300, 300, 4, 2, 32, 32, False, 4.0, (-12, 9)),
    (257, 257, 2, 1, 128, 0, True, 5.0, (-10, 10)), (1100, 1100, 2, 2, 64, 16, True, 1.0, (-13, 8)),
    (90, 1600, 2, 2, 128, 32, False, 0.2, (-13, -9)), (130, 64, 2, 2, 40, 8, False, 6.0, (-8, 10)),
    (520, 130, 6, 1, 64, 0, False, 8.0, (-12, 8)),
]


@pytest.mark.parametrize("lq,lk,h,hk,d,buckets,causal,sharp,sizes", CASES)
def test_values_of_all_sizes(eng, lq, lk, h, hk, d, buckets, causal, sharp, sizes):
    """Rows of dout, and blocks of values, of very different sizes beside each other, element by element."""
    print("sizes", lq, lk, h, hk, d, buckets, causal, sharp, sizes, flush=True)
    g = torch.Generator().manual_seed(91)

    def rand(*shape):
        return torch.randn(*shape, generator=g)

    q, k, v = (rand(1, lq, h, d) * sharp).to(F16), rand(1, lk, hk, d).to(F16), rand(1, lk, hk, d)
    v = (v * torch.exp2(-3 * (torch.arange(lk) // 64 % 3 == 0).float())[None, :, None, None]).to(F16)
    lo, hi = sizes
    do = (rand(1, lq, h, d) * torch.exp2((lo + (hi - lo) * torch.rand(lq, generator=g)).round())[None, :, None, None]).to(F16)
    table = rand(buckets, h).to(F16) if buckets else None
    scale = 0.25 / math.sqrt(d)  # (results within float16's range)
    more = dict(causal=causal, max_distance=100)
    got = gradients(q, k, v, do, table, scale, **more)
    want, bounds = grad_bounds(do.double(), q.double(), k.double(), v.double(), scale, F16,
                               table=None if table is None else table.double(), lift=LIFT, **more)
    for name, a, r, t in zip(("dq", "dk", "dv", "dtable"), got, want, bounds):
        if r is not None:
            big = r.abs() > 65000  # past float16's range, or at its end
            o.within(torch.where(big, torch.zeros_like(r), a.double().cpu()), torch.where(big, torch.zeros_like(r), r), t, name)
