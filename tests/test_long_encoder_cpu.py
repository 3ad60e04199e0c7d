"""What windowed attention, the gated product and products of 8-bit whole numbers promise that needs
no GPU: structures and codes as the header's, refusals before any launch, the oracle itself."""

from __future__ import annotations

import ctypes
import math
import re
import subprocess
from pathlib import Path

import pytest
import torch

import encoder_oracle as o
import long_encoder_oracle as lo
from cuda_vector_search import _ext, encoder

REPO = Path(__file__).resolve().parents[1]


def test_window_structure_and_codes_are_the_headers(tmp_path):
    names = [f[0] for f in _ext.AttentionWindow._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "cvs.h"\nint main(void) { printf("%zu", sizeof(cvs_attention_window));\n'
                   + "".join(f'printf(" %zu", offsetof(cvs_attention_window, {n}));\n' for n in names) + "return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_ext.AttentionWindow)] + [getattr(_ext.AttentionWindow, n).offset for n in names]
    d = dict(re.findall(r"#define\s+(CVS_ACT_[A-Z]+)\s+(\d+)", (REPO / "include" / "cvs.h").read_text()))
    assert encoder.GATES == {**encoder.ACTIVATIONS, "silu": int(d["CVS_ACT_SILU"]), "sigmoid": int(d["CVS_ACT_SIGMOID"])}


def test_tensors_off_the_gpu_are_refused():
    x, w = torch.zeros(2, 16, dtype=torch.float16), torch.zeros(8, 16, dtype=torch.float16)
    q = x.view(1, 2, 1, 16)
    values, scales = torch.zeros(8, 16, dtype=torch.int8), torch.zeros(8)
    for call in (lambda: encoder.gated_linear(x, w, w), lambda: encoder.gated_linear_backward(x, x, w, w, x),
                 lambda: encoder.quantize_rows(x), lambda: encoder.linear_int8(x, values, scales),
                 lambda: encoder.attention(q, q, q, window=1, sinks=1)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_windows_that_are_none_are_refused():
    q = torch.zeros(1, 2, 1, 16, dtype=torch.float16)
    for more, error in (({"sinks": 1}, RuntimeError), ({"window": -1}, RuntimeError), ({"window": (1, -1)}, RuntimeError),
                        ({"window": 1, "sinks": -2}, RuntimeError), ({"window": 1.0}, TypeError), ({"window": (1, 2, 3)}, ValueError),
                        ({"window": "ab"}, TypeError), ({"window": 1, "sinks": None}, TypeError)):
        with pytest.raises(error):
            encoder.attention(q, q, q, **more)


def test_entry_points_refuse_what_no_kernel_takes():
    """Checks that come before the device is asked for anything: on a machine without one, that is what refuses."""
    lib = _ext.open_library()
    a = _ext.AttentionArgs(batch=1, q_len=8, k_len=8, heads=1, k_heads=1, width=16, scale=1.0)
    out = ctypes.c_int64(-1)
    assert lib.cvs_attention_window_plan(ctypes.byref(a), None, 0, 0, ctypes.byref(out)) != 0
    assert b"null window" in lib.cvs_last_error()
    assert lib.cvs_attention_window_forward(ctypes.byref(a), None, None, None, None, 0, 0, None) != 0
    assert lib.cvs_attention_window_backward(ctypes.byref(a), None, None, None, None, None, None, None, None, None, None, 0, 0, None) != 0
    assert out.value == -1


def test_oracle_gradients_are_autograds():
    g = torch.Generator().manual_seed(0)

    def t(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()

    x, wg, wu, bg, bu, dy = t(5, 12), t(7, 12), t(7, 12), t(7), t(7), t(5, 7)
    for act in encoder.GATES:
        y, pre = lo.gated(x, wg, wu, bg, bu, act)
        for a, r in zip(lo.gated_grads(dy, x, wg, wu, pre, act), torch.autograd.grad(y, (x, wg, wu, bg, bu), dy)):
            assert torch.allclose(a, r)
    for causal, kl, ql, window in ((False, None, None, (2, 1, 1)), (True, [9, 0], None, (3, 0, 2)), (False, [4, 9], [9, 3], (0, 3, 0)),
                                   (True, None, None, (0, 0, 0)), (False, None, None, (9, 9, 9))):
        q, k, v, table, do = t(2, 9, 4, 8), t(2, 9, 2, 8), t(2, 9, 2, 8), t(8, 4), t(2, 9, 4, 8)
        more = dict(causal=causal, max_distance=6)
        more |= {} if kl is None else {"key_lengths": torch.tensor(kl)}
        more |= {} if ql is None else {"query_lengths": torch.tensor(ql)}
        got = lo.window_attention(q, k, v, do, 0.3, torch.bfloat16, *window, table, **more)
        want = torch.autograd.grad(torch.nan_to_num(got["out"][0]), (q, k, v, table), do)
        for name, r in zip(("dq", "dk", "dv", "dtable"), want):
            assert torch.allclose(got[name][0], torch.nan_to_num(r), atol=1e-12), name


def test_oracle_window_is_attention_where_nothing_is_hidden():
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(1, 20, 2, 16, generator=g, dtype=torch.float64) for _ in range(4))
    for causal in (False, True):
        want = o.attention(q, k, v, 0.25, causal=causal)
        for window in ((19, 19, 0), (0, 0, 20)):
            got = lo.window_attention(q, k, v, do, 0.25, torch.float16, *window, causal=causal)
            assert torch.allclose(got["out"][0], want[0]) and torch.allclose(got["lse"][0], want[1])
    hidden = lo.window_attention(q, k, v, do, 0.25, torch.float16, 3, 2, 1)["out"][0]
    assert not torch.allclose(hidden, o.attention(q, k, v, 0.25)[0])


def test_oracle_bounds_hold_rounded_results_and_no_planted_errors():
    g = torch.Generator().manual_seed(2)
    x, wg, wu = (torch.randn(*s, generator=g).half().double() for s in ((40, 64), (24, 64), (24, 64)))
    args = (x, wg * 0.125, wu * 0.125, None, None, "silu")
    (y, pre), (bound, _) = lo.gated(*args), lo.gated_bounds(*args, torch.float16)
    o.within(y.half(), y, bound, "y")
    with pytest.raises(AssertionError):
        o.within((y * (1 + 4 * o.U[torch.float16])).half(), y, bound, "y")
    with pytest.raises(AssertionError):
        o.within(lo.gated(x, wg * 0.125, wu * 0.125, None, None, "gelu")[0].half(), y, bound, "y")
    values, unit = lo.quantize(wg)
    args = (x, values, unit, None, None, None)
    want, tol = lo.linear_int8(*args)[0], lo.linear_int8_bounds(*args, torch.float16)
    o.within(want.half(), want, tol, "y")
    with pytest.raises(AssertionError):  # one whole number off by one
        values[3, 5] += 1
        o.within(lo.linear_int8(*args)[0].half(), want, tol, "y")
    q, k, v, do = (torch.randn(1, 30, 1, 16, generator=g).half().double() for _ in range(4))
    want = lo.window_attention(q, k, v, do, 0.25, torch.float16, 5, 4, 2)
    for name, window in (("out", (5, 4, 1)), ("out", (4, 4, 2)), ("dk", (5, 3, 2)), ("dv", (5, 4, 3)), ("dq", (6, 4, 2))):
        o.within(want[name][0].half(), *want[name], name)
        with pytest.raises(AssertionError):
            o.within(lo.window_attention(q, k, v, do, 0.25, torch.float16, *window)[name][0].half(), *want[name], name)


def test_oracle_rows_in_whole_numbers():
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5, 126.4, -0.49], [0.0] * 6, [1.0, math.nan, 0, 0, 0, 0], [2.0, -1.0, 1 / 127, 0, 0, 0]]).double()
    values, unit = lo.quantize(x)
    assert values[0].tolist() == [127, 0, 2, -2, 126, 0] and unit[0] == 1
    assert not values[1].any() and unit[1] == 0 and not values[2].any() and math.isnan(unit[2])
    assert values[3].tolist() == [127, -64, 0, 0, 0, 0]
