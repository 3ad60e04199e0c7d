"""Arguments of the encoder operators at the ends of what they take (needs an MI355X)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import encoder_oracle as o
from cuda_vector_search import _ext, encoder

pytestmark = pytest.mark.gpu

F16 = torch.float16


def half(*shape):
    return torch.randn(*shape, device="cuda").to(F16)


def test_a_scale_changed_in_place_counts(eng):
    """A scale, or a flag, held in a tensor is read at every call."""
    q, k, v = half(1, 40, 2, 32), half(1, 40, 2, 32), half(1, 40, 2, 32)
    scale, causal = torch.tensor(0.5), torch.tensor(True)
    for s, c in ((0.5, True), (0.0625, True), (0.0625, False), (0.25, True)):
        scale.fill_(s), causal.fill_(c)
        out, lse = encoder.attention_forward(q, k, v, scale=scale, causal=causal)
        want, want_lse = encoder.attention_forward(q, k, v, scale=s, causal=c)
        assert torch.equal(out, want) and torch.equal(lse, want_lse), f"scale {s}, causal {c}"
        for a, b in zip(encoder.attention_backward(v, q, k, v, out, lse, scale=scale, causal=causal)[:3],
                        encoder.attention_backward(v, q, k, v, out, lse, scale=s, causal=c)[:3]):
            assert torch.equal(a, b), f"gradient, scale {s}, causal {c}"


def plan(name, *sizes):
    """(status, workspace bytes) of a plan entry: no launch."""
    out = ctypes.c_int64(-1)
    rc = getattr(_ext.load().lib, name)(*sizes, 0, ctypes.byref(out))
    return rc, out.value


def test_linear_rows_that_no_launch_takes(eng):
    """2^31 - 256 rows and more are refused before a tile's last row passes an int; so are
    sizes whose tiles are 2^32 threads; the ones below have plans."""
    for m in (2**31 - 2, 2**31 - 255, 2**31 - 257):  # (the last: 2^23 tiles of 512 threads)
        assert plan("cvs_linear_plan", m, 8, 8)[0] != 0 and "rows" in str(_ext.load()._error(1))
        assert plan("cvs_linear_backward_plan", m, 8, 8, 0)[0] != 0
    for m in (2**31 - 2**12, 2**30 + 5, 2**24):
        rc, size = plan("cvs_linear_plan", m, 8, 8)
        assert rc == 0 and size == 0
        assert plan("cvs_linear_backward_plan", m, 8, 8, 0)[0] == 0


def test_linear_of_two_to_the_thirty_rows(eng):
    """Offsets past 2^32 in either matrix: the last rows, and some before, against the same rows alone."""
    m = 2**30 + 5
    x = torch.randn(m, 8, device="cuda", dtype=F16)
    w = half(8, 8)
    y = encoder.linear(x, w)
    dx = encoder.linear_backward(x, x, w, needs=(True, False, False))[0]
    for at in (0, 2**29 - 70, 2**30 - 100, m - 333):
        rows = x[at:at + 333].contiguous()
        assert torch.equal(y[at:at + 333], encoder.linear(rows, w))
        assert torch.equal(dx[at:at + 333], encoder.linear_backward(rows, rows, w, needs=(True, False, False))[0])
        assert torch.allclose(y[at:at + 333].float(), rows.float() @ w.float().T, atol=2e-2, rtol=1e-2)


def test_scales_that_fp32_cannot_divide_by(eng):
    """A bias is held divided by the scale: where that is infinite the call was answered with NaN."""
    q, k, v = half(1, 40, 2, 32), half(1, 40, 2, 32), half(1, 40, 2, 32)
    table = half(8, 2)
    for scale in (1e-45, 1e-300, 2.0**-101, 1e38, math.inf, -1.0):
        with pytest.raises(RuntimeError, match="scale"):
            encoder.attention(q, k, v, table, scale=scale, max_distance=9)
    ref = dict(table=table.double().cpu(), max_distance=9)
    args = [t.double().cpu() for t in (q, k, v)]
    out, lse = encoder.attention_forward(q, k, v, table, scale=2.0**-100, max_distance=9)
    o.within(out, o.attention(*args, 2.0**-100, **ref)[0], o.attention_bounds(*args, 2.0**-100, F16, **ref)[0], "out")
    grads = encoder.attention_backward(v, q, k, v, out, lse, table, scale=2.0**-100, max_distance=9)
    for a, r, b in zip(grads, o.attention_grads(args[2], *args, 2.0**-100, **ref),
                       o.attention_grad_bounds(args[2], *args, 2.0**-100, F16, **ref)):
        o.within(a, r, b, "gradient")


def test_plans_without_a_place_for_the_size(eng):
    """As the search's plans: a null pointer asks only whether there is a plan."""
    lib = _ext.load().lib
    assert lib.cvs_layer_norm_backward_plan(100, 64, 0, 0, None) == 0
    assert lib.cvs_linear_plan(100, 64, 64, 0, None) == 0
    assert lib.cvs_linear_backward_plan(100, 64, 64, 1, 0, None) == 0
    a = _ext.AttentionArgs(batch=1, q_len=8, k_len=8, heads=1, k_heads=1, width=16, scale=1.0)
    assert lib.cvs_attention_plan(ctypes.byref(a), 0, 0, None) == 0
    assert lib.cvs_attention_plan(ctypes.byref(a), 1, 0, None) == 0
    assert lib.cvs_attention_plan(None, 1, 0, None) != 0
