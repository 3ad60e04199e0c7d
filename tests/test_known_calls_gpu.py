"""Calls of sizes and strides that were seen before, of tensors that do not start on 16 bytes as the first ones did
(needs an MI355X)."""

from __future__ import annotations

import pytest
import torch

from cuda_vector_search import encoder

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def moved(t):
    """The same values, shape and strides, an element further on in memory than 16 bytes allow."""
    size = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    field = torch.zeros(size + 17, dtype=t.dtype, device=t.device)
    field = field[(-field.data_ptr() // t.element_size()) % 16 + 1:]
    other = field.as_strided(t.shape, t.stride())
    other.copy_(t)
    assert other.data_ptr() % 16 != 0 and other.stride() == t.stride()
    return other


def hold(call, operands):
    """call(*operands), and again with each operand moved, with all, and as first: the same values each time."""
    encoder._known.clear()
    want = call(*operands)
    assert len(encoder._known) == 1
    for at in range(len(operands) + 1):
        if at < len(operands) and operands[at] is None:
            continue
        others = [moved(t) if t is not None and at in (n, len(operands)) else t for n, t in enumerate(operands)]
        for args in (others, operands):
            assert all(a is b is None or torch.equal(a, b) for a, b in zip(call(*args), want)), at
    encoder._known.clear()
    others = [None if t is None else moved(t) for t in operands]  # not known from these
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(call(*others), want)) and not encoder._known
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(call(*operands), want)) and len(encoder._known) == 1


@pytest.mark.parametrize("m,k,n", [(1, 64, 24), (33, 136, 200), (300, 72, 264)])
def test_gated_linear_of_a_known_form(eng, m, k, n):
    def t(*shape):
        return torch.randn(*shape, device="cuda").to(BF16)

    for x in (t(m, k), t(m, k + 8)[:, :k], t(m, 1, k)):
        for bias in (None, t(n)):
            hold(lambda *a: encoder.gated_linear_forward(*a, keep_pre=True), (x, t(n, k), t(n, k), bias, t(n)))


@pytest.mark.parametrize("m,k,n", [(1, 64, 24), (33, 144, 200), (300, 80, 264)])
def test_linear_int8_of_a_known_form(eng, m, k, n):
    def t(*shape):
        return torch.randn(*shape, device="cuda").to(F16)

    for x in (t(m, k), t(m, k + 8)[:, :k], t(m, 1, k)):
        values, scales = encoder.quantize_rows(t(n, k))
        for bias, residual in ((None, None), (t(n), t(*x.shape[:-1], n))):
            hold(lambda x, v, s, b, r: (encoder.linear_int8(x, v, s, b, "gelu", r),), (x, values, scales, bias, residual))
        wide = t(m, n + 16)[:, 8:-8].reshape(*x.shape[:-1], n) if x.dim() == 3 else t(m, n + 16)[:, 8:-8]
        hold(lambda x, v, s, b, r: (encoder.linear_int8(x, v, s, b, None, r),), (x, values, scales, t(n), wide))
