"""Products of 8-bit whole numbers against their 64-bit plain form (needs an MI355X).

No counterpart in the reference.  Rows in whole numbers are held to the definition exactly, products
to bounds derived in long_encoder_oracle.
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


@pytest.mark.parametrize("rows,k,dtype", [(1, 16, F16), (5, 48, BF16), (130, 768, F16), (3, 1040, BF16), (7, 2048, F16), (2, 4096, BF16),
                                          (3, 4112, F16), (2, 131072, BF16)])
def test_quantize_rows(eng, rows, k, dtype):
    say("quantize", rows, k, dtype)
    x, xd = rand((rows, k), 71, dtype, 2.0, 0.3)
    values, scales = encoder.quantize_rows(x)
    want, unit = lo.quantize(xd)
    assert torch.equal(values.cpu(), want.to(torch.int8)) and torch.equal(scales.cpu(), unit.float())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_quantize_rows_at_ties_and_both_ends(eng, dtype):
    """Every quotient n + 1/2 goes to the even number; rows of subnormals and of the largest values keep the rule."""
    n = torch.arange(-127, 127).double()
    rows = []
    for top in (127.0, 254.0, 127 * 2.0**-10, 127 * 2.0**8):
        rows.append(torch.cat([torch.tensor([top, -top]), (n + 0.5) * (top / 127)]))
    rows.append(rows[0] * 0)
    big = torch.finfo(dtype).max
    rows.append(torch.linspace(-1, 1, 256).double() * big)
    small = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the smallest subnormal
    rows.append((torch.arange(256) % 7 - 3).double() * small)
    rows.append((torch.arange(256) - 128).double() * small)
    x = torch.stack(rows).to(dtype)
    ties = (x.double() * 127 / x.double().abs().amax(1, keepdim=True).clamp(min=1e-300)) % 1 == 0.5
    assert int(ties[:4].sum()) >= 4 * 200
    values, scales = encoder.quantize_rows(x.cuda())
    want, unit = lo.quantize(x.double())
    assert torch.equal(values.cpu(), want.to(torch.int8)) and torch.equal(scales.cpu(), unit.float())


def test_quantize_rows_of_every_pair(eng):
    """All float16 magnitudes against some largest ones: no quotient is rounded the wrong way."""
    every = torch.arange(0, 0x7c00, dtype=torch.int16).view(F16)
    for top in (0x0001, 0x0003, 0x03ff, 0x0401, 0x2e67, 0x3c01, 0x3fff, 0x7bff):
        value = torch.tensor([top], dtype=torch.int16).view(F16)
        fit = every[every <= value]
        fit = fit[-8192:]
        x = torch.cat([value, fit, fit.new_zeros(-(len(fit) + 1) % 16)])[None]
        values, _ = encoder.quantize_rows(x.cuda())
        assert torch.equal(values.cpu(), lo.quantize(x.double())[0].to(torch.int8)), hex(top)


def test_quantize_rows_not_finite_zero_and_views(eng):
    x, _ = rand((6, 64), 72, F16)
    want = encoder.quantize_rows(x)
    x[1, 3], x[2, 0], x[4, 63], x[5] = math.nan, math.inf, -math.inf, 0.0
    values, scales = encoder.quantize_rows(x)
    assert torch.isnan(scales[[1, 2, 4]]).all() and not values[[1, 2, 4, 5]].any() and scales[5] == 0
    for i in (0, 3):
        assert torch.equal(values[i], want[0][i]) and scales[i] == want[1][i]
    big, bigd = rand((3, 40, 300), 73, BF16)
    for view in (lambda t: t[:, :, 8:200], lambda t: t[:, 1, 1:33], lambda t: t[:, :, :96:2], lambda t: t[0, 0, :16], lambda t: t[:, :0, :16]):
        values, scales = encoder.quantize_rows(view(big))
        if values.numel():
            q, unit = lo.quantize(view(bigd))
            assert torch.equal(values.cpu(), q.to(torch.int8)) and torch.equal(scales.cpu(), unit.float())
        assert values.shape == view(big).shape and scales.shape == view(big).shape[:-1]


# sizes that take each tile, whole and in parts
SIZES = [(1, 16, 8, None, F16), (1, 768, 2048, "gelu", F16), (3, 4096, 72, "tanh", BF16), (23, 384, 1536, "gelu", F16), (32, 2048, 200, "relu", F16),
         (33, 2048, 200, "relu", F16), (16, 8192, 640, None, BF16), (65, 144, 136, "tanh", F16), (300, 768, 104, "gelu", BF16),
         (404, 3728, 1240, None, F16), (2049, 272, 1000, "gelu", F16), (6478, 64, 1752, "gelu", BF16), (8486, 64, 912, "tanh", F16),
         (1000, 4112, 64, None, BF16), (2, 131072, 16, None, F16),
         # the most rows and depth of one launch, and past them
         (32, 1792, 200, "gelu", BF16), (31, 1040, 72, None, F16), (14, 4112, 40, "relu", F16), (29, 2048, 64, None, BF16), (32, 16, 8, "tanh", F16)]


@pytest.mark.parametrize("m,k,n,act,dtype", SIZES)
def test_linear_int8(eng, m, k, n, act, dtype):
    say("int8", m, k, n, act, dtype)
    x, xd = rand((m, k), 81, dtype, 1.0, 0.1)
    w, _ = rand((n, k), 82, dtype, 1 / math.sqrt(k))
    b, bd = rand((n,), 83, dtype, 0.3)
    res, rd = rand((m, n), 84, dtype)
    values, scales = encoder.quantize_rows(w)
    vd, sd = values.double().cpu(), scales.double().cpu()
    y = encoder.linear_int8(x, values, scales, b, act, res)
    args = (xd, vd, sd, bd, act, rd)
    o.within(y, lo.linear_int8(*args)[0], lo.linear_int8_bounds(*args, dtype), "y")
    assert torch.equal(y, encoder.linear_int8(x, values, scales, b, act, res))
    args = (xd, vd, sd, None, act, None)
    o.within(encoder.linear_int8(x, values, scales, activation=act), lo.linear_int8(*args)[0], lo.linear_int8_bounds(*args, dtype), "y bare")


def test_linear_int8_is_near_the_product_it_stands_for(eng):
    """Rounding to 8 bits leaves about a hundredth of the result's size."""
    x, xd = rand((70, 512), 85, F16)
    w, wd = rand((256, 512), 86, F16, 512**-0.5)
    y = encoder.linear_int8(x, *encoder.quantize_rows(w)).double().cpu()
    want = xd @ wd.T
    # an operand's rounding is at most half a unit, of some 3.5 / 127: sqrt(1/12) of a unit on average, two of them
    assert float((y - want).norm() / want.norm()) < 2 * 3.8 / 127 / math.sqrt(12)


def test_linear_int8_largest_sums(eng):
    """Sums at the end of 32 bits: k = 2^17 of 127 * -128."""
    k = 1 << 17
    x = torch.full((2, k), 3.0, device="cuda", dtype=F16)
    x[1] *= -1
    values = torch.full((8, k), -128, device="cuda", dtype=torch.int8)
    values[1::2] = 127
    scales = torch.full((8,), 2.0**-20, device="cuda")
    y = encoder.linear_int8(x, values, scales).double().cpu()
    want = x.double().cpu()[:, :1] * k * values[:, 0].double().cpu() * 2.0**-20
    assert float((y - want).abs().max()) <= float((want * (o.U[F16] + 8 * o.F32)).abs().max())


def test_linear_int8_strides_shapes_and_odd_rows(eng):
    big, bigd = rand((6, 40, 600), 87, F16)
    w, _ = rand((72, 192), 88, F16, 0.1)
    values, scales = encoder.quantize_rows(w)
    vd, sd = values.double().cpu(), scales.double().cpu()
    for view in (lambda t: t[:, :, 104:296], lambda t: t[:, 2, 1:193], lambda t: t[:, :, :384:2], lambda t: t[3:4, :, 8:200],
                 lambda t: t[:, :1, 8:200].expand(6, 4, 192), lambda t: t[0, 0, :192]):
        args = (view(bigd), vd, sd, None, "gelu", None)
        o.within(encoder.linear_int8(view(big), values, scales, activation="gelu"), lo.linear_int8(*args)[0],
                 lo.linear_int8_bounds(*args, F16), "a view")
    x = big[0, :, :192].contiguous()
    want = encoder.linear_int8(x, values, scales)
    turned = values.t().contiguous().t()
    assert torch.equal(encoder.linear_int8(x, turned, scales.repeat_interleave(2)[::2]), want)
    bias = torch.randn(72, device="cuda").to(F16)
    x[1, 4], x[3, 9], x[5] = math.nan, math.inf, 0.0
    y = encoder.linear_int8(x, values, scales, bias)
    keep = [i for i in range(40) if i not in (1, 3, 5)]
    assert torch.isnan(y[[1, 3]]).all() and torch.equal(y[5], bias)
    assert torch.equal(y[keep], encoder.linear_int8(x[keep], values, scales, bias))
    assert encoder.linear_int8(x[:0], values, scales, bias).shape == (0, 72)


def test_linear_int8_reads_nothing_outside(eng):
    field = torch.full((79, 160), math.nan, device="cuda", dtype=BF16)
    field[1:-1, 8:-8] = torch.randn(77, 144, device="cuda").to(BF16)
    x = field[1:-1, 8:-8]
    values, scales = encoder.quantize_rows(torch.randn(200, 144, device="cuda").to(BF16))
    y = encoder.linear_int8(x, values, scales)
    assert torch.isfinite(y).all() and torch.equal(y, encoder.linear_int8(x.contiguous(), values, scales))
    for rows in (1, 16, 31):
        assert torch.equal(encoder.linear_int8(x[:rows], values, scales), y[:rows])


def test_int8_refusals(eng):
    def t(*shape, dtype=F16):
        return torch.randn(*shape, device="cuda").to(dtype)

    x, v = t(4, 32), torch.zeros(24, 32, device="cuda", dtype=torch.int8)
    s = torch.ones(24, device="cuda")
    for call, reason in (
        (lambda: encoder.quantize_rows(x.float()), "bfloat16"),
        (lambda: encoder.quantize_rows(t(4, 24)), "multiple of 16"),
        (lambda: encoder.quantize_rows(x.cpu()), "CUDA"),
        (lambda: encoder.linear_int8(x.float(), v, s), "bfloat16"),
        (lambda: encoder.linear_int8(x, v.to(torch.uint8), s), "int8"),
        (lambda: encoder.linear_int8(x, v[:, :16], s), "as wide"),
        (lambda: encoder.linear_int8(t(4, 24), v[:, :24], s), "multiple of 16"),
        (lambda: encoder.linear_int8(x, v[:20], s[:20]), "multiple of 8"),
        (lambda: encoder.linear_int8(x, v, s[:16]), "scales"),
        (lambda: encoder.linear_int8(x, v, s.half()), "float32"),
        (lambda: encoder.linear_int8(x, v, s, t(16)), "bias"),
        (lambda: encoder.linear_int8(x, v, s, residual=t(4, 16)), "residual"),
        (lambda: encoder.linear_int8(x.requires_grad_(), v, s), "no_grad"),
        (lambda: encoder.quantize_rows(x.requires_grad_()), "no_grad"),
    ):
        with pytest.raises(RuntimeError, match=reason):
            call()
    with pytest.raises(ValueError, match="activation"):
        encoder.linear_int8(t(4, 32), v, s, activation="silu")
    with torch.no_grad():
        assert encoder.linear_int8(x, v, s).shape == (4, 24)


def workspace(m, k, n):
    import ctypes

    from cuda_vector_search import _ext

    out = ctypes.c_int64(-1)
    assert _ext.load().lib.cvs_linear_int8_plan(m, k, n, 0, ctypes.byref(out)) == 0
    return out.value


def test_linear_int8_few_rows_take_one_launch_where_it_is_the_faster(eng):
    """Every workgroup of the one launch takes all rows: not for outputs of more columns than the CUs take at once, nor for
    more rows than it was found faster for.  (Only the tiles have a workspace.)"""
    for m, k, n in ((1, 768, 2048), (23, 384, 1536), (32, 1024, 8192), (16, 1024, 16384), (16, 1920, 8192), (28, 2048, 8192)):
        assert workspace(m, k, n) == 0, (m, k, n)
    for m, k, n in ((1, 768, 131072), (8, 768, 32768), (32, 1792, 4096), (24, 1280, 512), (8, 2048, 16384), (29, 2048, 512), (1, 2064, 64), (33, 64, 64)):
        assert workspace(m, k, n) > 0, (m, k, n)


@pytest.mark.parametrize("m,k,n", [(1, 64, 131072), (16, 1024, 16384), (17, 1024, 16384), (28, 2048, 264), (29, 2048, 264), (16, 1040, 8192),
                                   (16, 1040, 8200), (2, 48, 1 << 20)])
def test_linear_int8_on_both_sides_of_the_rule(eng, m, k, n):
    say("int8 rule", m, k, n)
    x, xd = rand((m, k), 91, F16)
    values, scales = encoder.quantize_rows(rand((n, k), 92, F16, 1 / math.sqrt(k))[0])
    args = (xd, values.double().cpu(), scales.double().cpu(), None, "tanh", None)
    o.within(encoder.linear_int8(x, values, scales, activation="tanh"), lo.linear_int8(*args)[0], lo.linear_int8_bounds(*args, F16), "y")
