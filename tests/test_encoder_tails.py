"""The slope of tanh keeps its digits where it is small (needs an MI355X)."""

from __future__ import annotations

import pytest
import torch

from cuda_vector_search import encoder

pytestmark = pytest.mark.gpu


def test_tanh_slope_far_out(eng):
    """1 / cosh^2 relative to itself: dz and dx are each rounded once to bfloat16, the slope's fp32 steps (its
    exponent of up to 60 with them) take less than 2^-16."""
    u = 2.0**-8
    z = torch.linspace(-20, 20, 1024).to(torch.bfloat16).view(64, 16)
    eye = torch.eye(16, dtype=torch.bfloat16, device="cuda")
    dy = torch.ones(64, 16, dtype=torch.bfloat16, device="cuda")
    dx, _, _ = encoder.linear_backward(dy, dy, eye, "tanh", z.cuda())
    want = torch.cosh(z.double()).pow(-2)
    off = ((dx.double().cpu() - want) / want).abs()
    assert float(off.max()) <= u + 2.0**-16, f"off by {float(off.max())} at {float(z.reshape(-1)[off.argmax()])}"
