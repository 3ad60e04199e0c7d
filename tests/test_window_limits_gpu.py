"""What windowed attention takes of many first keys (needs an MI355X)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import encoder_oracle as o
from cuda_vector_search import _ext, encoder

pytestmark = pytest.mark.gpu


def plan(backward, batch, heads, k_heads, k_len, sinks):
    """Whether the plan of a call of one row a sequence is made (nothing is launched)."""
    a = _ext.AttentionArgs(batch=batch, q_len=1, k_len=k_len, heads=heads, k_heads=k_heads, width=64, scale=1.0)
    size, lib = ctypes.c_int64(-1), _ext.load().lib
    rc = lib.cvs_attention_window_plan(ctypes.byref(a), ctypes.byref(_ext.AttentionWindow(1, 1, sinks)), backward, 0, ctypes.byref(size))
    assert (rc == 0) == (size.value >= 0)
    if rc != 0:
        assert b"first keys" in lib.cvs_last_error()
    return rc == 0


def test_many_first_keys_are_refused_by_a_backward_pass_only(eng):
    for batch, heads, k_heads in ((1024, 1, 1), (16, 64, 64), (16, 64, 1)):
        assert plan(0, batch, heads, k_heads, 65536, 65536) and plan(1, batch, heads, k_heads, 65536, 65536)
    most = 8191 * 128  # keys: the most of 1024 heads
    assert plan(0, 1024, 1, 1, most, most) and not plan(1, 1024, 1, 1, most, most)
    assert plan(1, 1024, 1, 1, most, 1 << 17) and plan(1, 16, 64, 1, most, most)


def test_many_first_keys_of_many_heads(eng):
    """Every key a first one, of 64 sequences of 64 heads: attention without a window."""
    g = torch.Generator(device="cuda").manual_seed(5)
    q, do = (torch.randn(64, 1, 64, 8, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    k, v = (torch.randn(64, 16384, 1, 8, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    results = []
    for more in ({"window": 0, "sinks": 1 << 20}, {}):
        out, lse = encoder.attention_forward(q, k, v, **more)
        results.append((out, *encoder.attention_backward(do, q, k, v, out, lse, **more)[:3]))
    for name, a, b in zip(("out", "dq", "dk", "dv"), *results):
        # each is within U of the exact value for each of its roundings (its own, p's or ds', out's in delta)
        assert float((a.double() - b.double()).norm()) <= 6 * o.U[torch.bfloat16] * float(b.double().norm()), name
