"""What calls of the long-context encoder's operators leave in a program's hands, on the CPU (the library that copies its
first operand takes the kernels' place)."""

from __future__ import annotations

import torch

from cuda_vector_search import encoder
from test_long_encoder_modes import N, PRE, WIDTH, half, stub  # noqa: F401 (stub: a fixture for every test)


def test_weights_gradients_have_memory_of_their_own():
    """Neither gated weight's gradient holds, or is lost with, the other's memory."""
    x, gate, up = half(N, WIDTH), half(WIDTH, WIDTH), half(WIDTH, WIDTH)
    for rows in (N, 0):
        _, dgate, dup, _, _ = encoder.gated_linear_backward(x[:rows], x[:rows], gate, up, PRE[:rows])
        for t in (dgate, dup):
            assert t.untyped_storage().nbytes() == t.numel() * t.element_size() and t.storage_offset() == 0
        assert dgate.untyped_storage().data_ptr() != dup.untyped_storage().data_ptr()
    gate.requires_grad_(), up.requires_grad_()
    encoder.gated_linear(x, gate, up).float().sum().backward()
    for t in (gate.grad, up.grad):
        assert t.untyped_storage().nbytes() == t.numel() * t.element_size()
