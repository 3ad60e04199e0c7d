"""What the encoder operators promise that needs no GPU: the C structure's layout, the
bucket rule, the entry points' refusals before any launch, the oracle itself."""

from __future__ import annotations

import ctypes
import math
import re
import subprocess
from pathlib import Path

import pytest
import torch

import encoder_oracle as o
from cuda_vector_search import _ext, encoder

REPO = Path(__file__).resolve().parents[1]


def test_attention_structure_is_the_headers(tmp_path):
    names = [f[0] for f in _ext.AttentionArgs._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "cvs.h"\nint main(void) { printf("%zu", sizeof(cvs_attention));\n'
                   + "".join(f'printf(" %zu", offsetof(cvs_attention, {n}));\n' for n in names) + "return 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_ext.AttentionArgs)] + [getattr(_ext.AttentionArgs, n).offset for n in names]


def test_codes_match_the_header():
    d = dict(re.findall(r"#define\s+(CVS_[A-Z_0-9]+)\s+(\d+)", (REPO / "include" / "cvs.h").read_text()))
    assert encoder.TYPES == {torch.float16: int(d["CVS_TYPE_F16"]), torch.bfloat16: int(d["CVS_TYPE_BF16"]),
                             torch.float32: int(d["CVS_TYPE_F32"])}
    assert encoder.ACTIVATIONS == {None: int(d["CVS_ACT_NONE"]), "gelu": int(d["CVS_ACT_GELU"]),
                                   "relu": int(d["CVS_ACT_RELU"]), "tanh": int(d["CVS_ACT_TANH"])}


def test_tensors_off_the_gpu_are_refused():
    x, w = torch.zeros(2, 16, dtype=torch.float16), torch.zeros(16, dtype=torch.float16)
    for call in (lambda: encoder.layer_norm(x, w), lambda: encoder.linear(x, torch.zeros(8, 16, dtype=torch.float16)),
                 lambda: encoder.attention(x.view(1, 2, 1, 16), x.view(1, 2, 1, 16), x.view(1, 2, 1, 16))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_bucket_rule():
    """32 buckets, both directions, to 128: single distances to 7, then 8-11, 12-15, 16-22, ... from 91 on."""
    found = o.bucket(torch.arange(-200, 201), 32, False, 128)
    past, future = found[:201].flip(0), found[200:]
    assert past[:8].tolist() == list(range(8))
    starts = [int((past == u).nonzero()[0]) for u in range(16)]
    assert starts[8:] == [8, 12, 16, 23, 32, 46, 64, 91]
    assert torch.equal(future[1:], past[1:] + 16)
    one = o.bucket(torch.arange(-200, 3), 32, True, 128)
    assert one[-3:].tolist() == [0, 0, 0] and int(one[0]) == 31


def test_oracle_gradients_are_autograds():
    """The oracle's formulas against torch's own derivatives, in 64 bits."""
    g = torch.Generator().manual_seed(0)

    def t(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()

    x, w, b, dy = t(5, 12), t(12), t(12), t(5, 12)
    y, mean, rstd = o.norm(x, w, b, 1e-5)
    for a, r in zip(o.norm_grads(dy, x, w, mean, rstd), torch.autograd.grad(y, (x, w, b), dy)):
        assert torch.allclose(a, r)
    lw, lb = t(7, 12), t(7)
    for act in (None, "gelu", "relu", "tanh"):
        y, z = o.linear(x, lw, lb, act, None)
        dy = t(5, 7)
        for a, r in zip(o.linear_grads(dy, x, lw, act, z), torch.autograd.grad(y, (x, lw, lb), dy)):
            assert torch.allclose(a, r)
    for causal, kl, ql in ((False, None, None), (True, [9, 0], None), (False, [4, 9], [9, 3])):
        q, k, v, table, do = t(2, 9, 4, 8), t(2, 9, 2, 8), t(2, 9, 2, 8), t(8, 4), t(2, 9, 4, 8)
        more = dict(causal=causal, max_distance=6)
        more |= {} if kl is None else {"key_lengths": torch.tensor(kl)}
        more |= {} if ql is None else {"query_lengths": torch.tensor(ql)}
        out, lse = o.attention(q, k, v, 0.3, table=table, **more)
        want = torch.autograd.grad(torch.nan_to_num(out), (q, k, v, table), do)
        for a, r in zip(o.attention_grads(do, q, k, v, 0.3, table, **more), want):
            assert torch.allclose(a, torch.nan_to_num(r), atol=1e-12)


def test_oracle_bounds_hold_rounded_results():
    """A result rounded once is inside each bound, a planted error of a few roundings is not."""
    g = torch.Generator().manual_seed(1)
    x, w = (torch.randn(40, 64, generator=g).half().double(), torch.randn(64, generator=g).half().double())
    y, bound = o.norm(x, w, None, 1e-5)[0], o.norm_bounds(x, w, None, 1e-5, torch.float16)[0]
    o.within(y.half(), y, bound, "y")
    with pytest.raises(AssertionError):
        o.within((y * (1 + 4 * o.U[torch.float16])).half(), y, bound, "y")
    q, k, v = (torch.randn(1, 30, 1, 16, generator=g).half().double() for _ in range(3))
    want, tol = o.attention(q, k, v, 0.25)[0], o.attention_bounds(q, k, v, 0.25, torch.float16)[0]
    o.within(want.half(), want, tol, "out")
    wrong = o.attention(q, k, v, 0.25, key_lengths=torch.tensor([29]))[0]
    with pytest.raises(AssertionError):
        o.within(wrong.half(), want, tol, "out")
    assert math.isinf(float(o.attention(q, k, v, 0.25, key_lengths=torch.tensor([0]))[1][0, 0, 0]))
