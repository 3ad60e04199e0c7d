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


def test_a_backward_pass_takes_the_forward_passes_scale_and_flag(monkeypatch):
    """Values held in tensors or other objects may have changed by then."""
    seen = []
    args = encoder._attention_args

    def record(q, k, v, bias_table, key_lengths, query_lengths, query_start, causal, scale, max_distance, win):
        seen.append((bool(causal), float(scale), int(max_distance), win))
        return args(q, k, v, bias_table, key_lengths, query_lengths, query_start, causal, scale, max_distance, win)

    monkeypatch.setattr(encoder, "_attention_args", record)
    x = half(N, WIDTH).view(1, N, 1, WIDTH).requires_grad_()
    scale, causal, window, distance = torch.tensor(0.25), torch.tensor(True), torch.tensor([2, 1]), torch.tensor(20)
    y = encoder.attention(x, x, x, half(4, 1), causal=causal, scale=scale, max_distance=distance, window=window, sinks=1)
    scale.fill_(0.5), causal.fill_(False), window.fill_(3), distance.fill_(30)
    y.float().sum().backward()
    assert len(seen) == 2 and seen[0] == seen[1] == (True, 0.25, 20, (2, 1, 1))
