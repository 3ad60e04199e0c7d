"""Arguments of the encoder operators at the ends of what they take (needs an MI355X)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

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
