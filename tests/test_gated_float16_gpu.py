"""The gated product's gradients in float16 keep their digits where the products' operand, dz = [dg, du], would be
subnormal or infinite as float16 numbers (needs an MI355X)."""

from __future__ import annotations

import math

import pytest
import torch

import encoder_oracle as o
import long_encoder_oracle as lo
from cuda_vector_search import encoder

pytestmark = pytest.mark.gpu

F16 = torch.float16
NAMES = ("dx", "dgate", "dup", "dgate_bias", "dup_bias")


def gradients(m, k, n, act, dy_size, factor=1.0, x_size=1.0, seed=91):
    """(the kernels' gradients, the formulas' in 64 bits) for factors of size ``factor``, weights of 1 / factor."""
    g = torch.Generator().manual_seed(seed)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(F16)

    x, dy, pre = rand(m, k, scale=x_size), rand(m, n, scale=dy_size), rand(m, 2 * n, scale=factor)
    gate, up = (rand(n, k, scale=1 / (factor * math.sqrt(k))) for _ in range(2))
    got = encoder.gated_linear_backward(*(t.cuda() for t in (dy, x, gate, up, pre)), act)
    return got, lo.gated_grads(*(t.double() for t in (dy, x, gate, up, pre)), act)


def hold(got, want, m, what):
    # By norm: a result rounded once (U / sqrt 3), of more than 32 rows dz's rounding as large, 8% for the luck of some 1000
    # values (as in test_gated_linear_gpu); the biases' sums are of values that were not rounded.  Beside them half
    # the spacing of the result's own subnormals, relative to its size.
    for name, a, r in zip(NAMES, got, want):
        a = a.double().cpu()
        if name.endswith("bias"):  # (sums of many rows, which may be past the type themselves)
            small = r.abs() < 65000
            a, r = a[small], r[small]
        assert torch.isfinite(a).all(), f"{what} {name} is not finite"
        roundings = 1 if m <= 32 or name.endswith("bias") else 2
        if r.numel() == 0:
            continue
        room = 1.08 * o.U[F16] * math.sqrt(roundings / 3) + 2.0**-25 / float(r.square().mean().sqrt())
        off = float((a - r).norm() / r.norm())
        assert off <= room, f"{what} {name}: {off} of {room}"


@pytest.mark.parametrize("power", [-18, -15, -12, -7, 0, 9])
@pytest.mark.parametrize("m,k,n,act", [(4096, 64, 64, "silu"), (2000, 136, 256, None), (20, 384, 256, "gelu"), (1, 512, 512, "sigmoid")])
def test_gradients_of_all_sizes(eng, m, k, n, act, power):
    """Gradients at both ends of float16's range; the rows' are small so that sums stay inside it."""
    print("gated gradients", m, k, n, act, power, flush=True)
    hold(*gradients(m, k, n, act, 2.0**power, x_size=2.0 ** (-6 if power > 0 else 0)), m, f"2^{power}")


@pytest.mark.parametrize("m", [3, 32, 33, 700])
def test_products_past_the_type_of_finite_results(eng, m):
    """dz past 65504, whose products with weights and rows below 1 are finite."""
    print("gated gradients past the type", m, flush=True)
    hold(*gradients(m, 128, 64, None, 2.0**9, factor=2.0**9, x_size=2.0**-10), m, "past the type")


def test_a_large_row_beside_small_ones(eng):
    """One row's gradients 2^20 times the others': its own results are whole, and the others' rows keep their digits."""
    g = torch.Generator().manual_seed(95)
    m, k, n = 200, 64, 64
    x, dy, pre = ((torch.randn(m, c, generator=g) * s).to(F16) for c, s in ((k, 1.0), (n, 2.0**-11), (2 * n, 1.0)))
    dy[77] = (torch.randn(n, generator=g) * 2.0**9).to(F16)
    gate, up = ((torch.randn(n, k, generator=g) / 8).to(F16) for _ in range(2))
    got = encoder.gated_linear_backward(*(t.cuda() for t in (dy, x, gate, up, pre)), "silu")
    want = lo.gated_grads(*(t.double() for t in (dy, x, gate, up, pre)), "silu")
    hold(got, want, m, "all")
    rest = torch.arange(m) != 77
    hold(got[:1], [want[0]], m, "all")
    hold([got[0][rest.cuda()]], [want[0][rest]], m, "the others")


@pytest.mark.parametrize("m", [8, 300])
def test_zero_and_not_finite_gradients(eng, m):
    """Nothing but zeros; and values that are not finite, which reach their own rows' dx only."""
    g = torch.Generator().manual_seed(97)
    k, n = 64, 72
    x, dy, pre = ((torch.randn(m, c, generator=g)).to(F16).cuda() for c in (k, n, 2 * n))
    gate, up = ((torch.randn(n, k, generator=g) / 8).to(F16).cuda() for _ in range(2))
    assert not any(t.any() for t in encoder.gated_linear_backward(torch.zeros_like(dy), x, gate, up, pre))
    for size in (2.0**-16, 1.0, 2.0**12):
        small = dy * size
        want = encoder.gated_linear_backward(small, x * 2.0**-6, gate, up, pre)[0]
        bad = small.clone()
        bad[2, 3], bad[5, 1] = math.inf, math.nan
        dx = encoder.gated_linear_backward(bad, x * 2.0**-6, gate, up, pre)[0]
        rows = torch.ones(m, dtype=torch.bool, device="cuda")
        rows[[2, 5]] = False
        assert not torch.isfinite(dx[2]).any() and torch.isnan(dx[5]).all()
        # (another row may hold the largest value, and decide the exponent)
        assert float((dx[rows].double() - want[rows].double()).norm()) <= 2 * o.U[F16] * float(want[rows].double().norm()) + 2.0**-25 * math.sqrt(m * k)


def test_gradients_replayed_from_a_graph(eng):
    """A captured pass takes the exponent of the values it is replayed with."""
    g = torch.Generator().manual_seed(99)
    for m in (16, 500):
        x, dy, pre = ((torch.randn(m, c, generator=g)).to(F16).cuda() for c in (64, 72, 144))
        gate, up = ((torch.randn(72, 64, generator=g) / 8).to(F16).cuda() for _ in range(2))
        first = dy.clone()
        encoder.gated_linear_backward(dy, x, gate, up, pre)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = encoder.gated_linear_backward(dy, x, gate, up, pre)
        for size in (1.0, 2.0**-17, 2.0**10, 2.0**-8, 1.0):
            dy.copy_(first * size)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, encoder.gated_linear_backward(dy, x, gate, up, pre)))
