"""The encoder operators where torch records or differentiates otherwise than by autograd's
backward pass: forward-mode derivatives, ``torch.jit.trace``, proxy tracing.

The kernels write through pointers, which none of these sees, so each call has to go through
an autograd function (which torch records, or refuses itself) or be refused.  The library is
replaced by one that copies its first operand, so that this runs without a GPU.
"""

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
            source, results = args[0], {"cvs_layer_norm": (8,), "cvs_linear": (11,), "cvs_attention_forward": (1,),
                                        "cvs_layer_norm_backward": (10,), "cvs_linear_backward": (11,),
                                        "cvs_attention_backward": (5, 6, 7)}[name]
            if name == "cvs_attention_forward":
                source = args[0]._obj.q
            elif name == "cvs_attention_backward":
                source = args[1]
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
    monkeypatch.setattr(encoder, "_calls", {})
    monkeypatch.setattr(encoder, "_plans", {})


def half(*shape):
    return torch.randn(*shape).half()


def heads(t):
    return t.view(1, N, 1, WIDTH)


OPERATORS = {
    "layer_norm": lambda x, w: encoder.layer_norm(x, w[0]),
    "linear": lambda x, w: encoder.linear(x, w, activation="gelu"),
    "attention": lambda x, w: encoder.attention(heads(x), heads(x), heads(x)),
}
STAT = torch.zeros(N)
PASSES = {
    "layer_norm_forward": lambda x, w: encoder.layer_norm_forward(x, w[0])[0],
    "layer_norm_backward": lambda x, w: encoder.layer_norm_backward(x, x, w[0], STAT, STAT)[0],
    "linear_forward": lambda x, w: encoder.linear_forward(x, w)[0],
    "linear_backward": lambda x, w: encoder.linear_backward(x, x, w)[0],
    "attention_forward": lambda x, w: encoder.attention_forward(heads(x), k=heads(x), v=heads(x))[0],
    "attention_backward": lambda x, w: encoder.attention_backward(heads(x), heads(x), heads(x), heads(x), out=heads(x),
                                                                  lse=torch.zeros(1, 1, N))[0],
}
CALLS = {**OPERATORS, **PASSES}


@pytest.mark.parametrize("name", CALLS)
def test_the_stub_copies(name):
    x, w = half(N, WIDTH), half(WIDTH, WIDTH)
    assert torch.equal(CALLS[name](x, w).reshape(N, WIDTH), x)


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    """No tangent may be dropped: every call with a dual tensor raises, one without still answers."""
    x, w = half(N, WIDTH), half(WIDTH, WIDTH)
    with fw.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward-mode"):
            CALLS[name](fw.make_dual(x, torch.ones_like(x)), w)
        if name != "attention" and not name.startswith("attention"):
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward-mode"):
                CALLS[name](x, fw.make_dual(w, torch.ones_like(w)))
        assert torch.equal(CALLS[name](x, w).reshape(N, WIDTH), x)


@pytest.mark.parametrize("name", CALLS)
def test_function_transforms_are_refused(name):
    x, w = half(N, WIDTH), half(WIDTH, WIDTH)
    for transform in (lambda: torch.func.jvp(lambda t: CALLS[name](t, w), (x,), (x,)),
                      lambda: torch.func.grad(lambda t: CALLS[name](t, w).float().sum())(x)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            transform()


@pytest.mark.parametrize("name", OPERATORS)
@pytest.mark.parametrize("grad", [False, True])
def test_traced_operators_compute(name, grad):
    """A traced call computes from its inputs, whether or not the example asked for gradients."""
    w = half(WIDTH, WIDTH)
    traced = torch.jit.trace(lambda t: OPERATORS[name](t, w), half(N, WIDTH).requires_grad_(grad), check_trace=False)
    for _ in range(3):
        x = half(N, WIDTH)
        assert torch.equal(traced(x).reshape(N, WIDTH), x)


@pytest.mark.parametrize("name", PASSES)
def test_traced_passes_are_refused(name):
    w = half(WIDTH, WIDTH)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: PASSES[name](t, w), half(N, WIDTH), check_trace=False)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_proxy_tracing_is_refused(name, grad):
    w = half(WIDTH, WIDTH)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda t: CALLS[name](t, w))(half(N, WIDTH).requires_grad_(grad))
