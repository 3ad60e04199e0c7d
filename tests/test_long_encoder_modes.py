"""Windowed attention, the gated product and products of 8-bit whole numbers where torch records or
differentiates otherwise than by autograd's backward pass (as test_encoder_modes, whose library that
copies its first operand takes the kernels' place, without a GPU)."""

from __future__ import annotations

import ctypes
import types

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

from cuda_vector_search import _ext, encoder

N, WIDTH = 4, 16  # every operand and result is N x WIDTH (attention: as [1, N, 1, WIDTH])


class CopyLibrary:
    """Results are copies of the first operand, plans need no workspace."""

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_plan"):
                args[-1]._obj.value = 0
                return 0
            results = {"cvs_gated_linear": (11,), "cvs_gated_linear_backward": (12,), "cvs_linear_int8": (12,), "cvs_quantize_rows": (),
                       "cvs_attention_window_forward": (2,), "cvs_attention_window_backward": (6, 7, 8)}[name]
            source = {"cvs_attention_window_forward": lambda: args[0]._obj.q, "cvs_attention_window_backward": lambda: args[2]}.get(name, lambda: args[0])()
            for at in results:
                if args[at] is not None:
                    ctypes.memmove(args[at], source, N * WIDTH * 2)
            return 0

        return call


@pytest.fixture(autouse=True)
def stub(monkeypatch):
    monkeypatch.setattr(encoder, "_tensor", lambda *a, **k: None)
    monkeypatch.setattr(_ext, "load", lambda verbose=False: types.SimpleNamespace(lib=CopyLibrary()))
    monkeypatch.setattr(_ext, "raw_stream", lambda device: 0)
    for cache in ("_calls", "_plans", "_known"):
        monkeypatch.setattr(encoder, cache, {})


def half(*shape):
    return torch.randn(*shape).half()


def heads(t):
    return t.view(1, N, 1, WIDTH)


VALUES, SCALES, PRE = torch.zeros(WIDTH, WIDTH, dtype=torch.int8), torch.zeros(WIDTH), torch.zeros(N, 2 * WIDTH).half()
WINDOW = dict(window=(2, 1), sinks=1)
OPERATORS = {
    "gated_linear": lambda x, w: encoder.gated_linear(x, w, w),
    "attention": lambda x, w: encoder.attention(heads(x), heads(x), heads(x), **WINDOW),
}
PASSES = {
    "gated_linear_forward": lambda x, w: encoder.gated_linear_forward(x, w, up=w)[0],
    "gated_linear_backward": lambda x, w: encoder.gated_linear_backward(x, x, w, w, PRE)[0],
    "attention_forward": lambda x, w: encoder.attention_forward(heads(x), k=heads(x), v=heads(x), **WINDOW)[0],
    "attention_backward": lambda x, w: encoder.attention_backward(heads(x), heads(x), heads(x), heads(x), out=heads(x),
                                                                  lse=torch.zeros(1, 1, N), **WINDOW)[0],
}
SERVING = {
    "linear_int8": lambda x, w: encoder.linear_int8(x, VALUES, scales=SCALES, residual=w[:N]),
    "quantize_rows": lambda x, w: encoder.quantize_rows(x),
}
CALLS = {**OPERATORS, **PASSES, **SERVING}


@pytest.mark.parametrize("name", {**OPERATORS, **PASSES, "linear_int8": 0})
def test_the_stub_copies(name):
    x, w = half(N, WIDTH), half(WIDTH, WIDTH)
    for _ in range(2):  # (checked, and known)
        assert torch.equal(CALLS[name](x, w).reshape(N, WIDTH), x)


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    """No tangent may be dropped: every call with a dual tensor raises, before and after the call is known."""
    x, w = half(N, WIDTH), half(WIDTH, WIDTH)
    for _ in range(2):
        with fw.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward-mode|derivative"):
                CALLS[name](fw.make_dual(x, torch.ones_like(x)), w)
            if not name.startswith("attention") and name != "quantize_rows":
                with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward-mode|derivative"):
                    CALLS[name](x, fw.make_dual(w, torch.ones_like(w)))
            CALLS[name](x, w)


@pytest.mark.parametrize("name", CALLS)
def test_function_transforms_are_refused(name):
    x, w = half(N, WIDTH), half(WIDTH, WIDTH)
    CALLS[name](x, w)
    for transform in (lambda: torch.func.jvp(lambda t: CALLS[name](t, w), (x,), (x,)),
                      lambda: torch.func.grad(lambda t: CALLS[name](t, w)[0].float().sum())(x)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            transform()


@pytest.mark.parametrize("name", SERVING)
def test_gradients_of_serving_calls_are_refused(name):
    x, w = half(N, WIDTH).requires_grad_(), half(WIDTH, WIDTH)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no_grad"):
            CALLS[name](x, w)
        with torch.no_grad():
            CALLS[name](x, w)


@pytest.mark.parametrize("name", OPERATORS)
@pytest.mark.parametrize("grad", [False, True])
def test_traced_operators_compute(name, grad):
    """A traced call computes from its inputs, whether or not the example asked for gradients."""
    w = half(WIDTH, WIDTH)
    traced = torch.jit.trace(lambda t: OPERATORS[name](t, w), half(N, WIDTH).requires_grad_(grad), check_trace=False)
    for _ in range(3):
        x = half(N, WIDTH)
        assert torch.equal(traced(x).reshape(N, WIDTH), x)


@pytest.mark.parametrize("name", {**PASSES, **SERVING})
def test_traced_passes_are_refused(name):
    w = half(WIDTH, WIDTH)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: CALLS[name](t, w), half(N, WIDTH), check_trace=False)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_proxy_tracing_is_refused(name, grad):
    w = half(WIDTH, WIDTH)
    CALLS[name](half(N, WIDTH), w)  # (known, too)
    with pytest.raises(RuntimeError, match="traced|derivative"):
        make_fx(lambda t: CALLS[name](t, w))(half(N, WIDTH).requires_grad_(grad))
