"""The layer of a text encoder: what makes the rows of an ``Index``, and what trains it.

The reference searches embeddings that a caller brings; it has no counterpart of
these operators.  Each runs hand-written gfx950 kernels (``libcvs_hip.so`` through
``_ext``) on the current stream of its tensors' GPU:

* ``layer_norm(x, weight, bias)``;
* ``linear(x, weight, bias, activation, residual)``, a matrix product with its epilogue;
* ``attention(q, k, v, ...)``, softmax attention over sequences of differing lengths,
  causal or not, with shared key heads and a learned bias by relative position.

These three are differentiable.  ``*_forward`` and ``*_backward`` are the passes
themselves, for programs that keep the saved tensors on their own.  Tensors are float16
or bfloat16 (``layer_norm``: float32 too), all of one type; results have it too, with
fp32 sums inside.  A refused argument raises ``RuntimeError`` with the reason; there
is no torch fallback.  Forward-mode derivatives and proxy tracing are refused too;
``torch.jit.trace`` records the three as Python calls.
"""

from __future__ import annotations

import ctypes
import functools
import math
import operator

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _ext

TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
ACTIVATIONS = {None: 0, "gelu": 1, "relu": 2, "tanh": 3}
_I64 = ctypes.c_int64
_I64x3 = _I64 * 3

_plans: dict = {}  # workspace bytes by operator and sizes (a pure function of them)


def _check(rc: int) -> None:
    if rc != 0:
        raise _ext.load()._error(rc)


_tracing = torch._C._get_tracing_state
_mode = torch._C._get_dispatch_mode
_PROXY = torch._C._TorchDispatchModeKey.PROXY


def _library():
    """The library, to be written with through pointers: not while torch's proxies record, which
    would see only the allocations (and replay those: results of memory nobody wrote)."""
    if _mode(_PROXY) is not None:
        raise RuntimeError("encoder operators cannot be traced by proxies")
    return _ext.load().lib


def _has_tangent(values) -> bool:
    """(Where forward_ad._current_level says that there may be any.)"""
    return any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in values)


def _bare(passes):
    """A pass of its own, which no autograd function announces to torch: refused where a trace
    records or a tensor carries a tangent.  ``.inner`` is the pass itself."""

    @functools.wraps(passes)
    def call(*args, **kwargs):
        if _tracing() is not None:
            raise RuntimeError(f"{passes.__name__} cannot be traced; {passes.__name__.rsplit('_', 1)[0]} can")
        if forward_ad._current_level >= 0 and _has_tangent((*args, *kwargs.values())):
            raise RuntimeError(f"{passes.__name__} has no forward-mode derivative")
        return passes(*args, **kwargs)

    call.inner = passes
    return call


def _through_autograd(*tensors) -> bool:
    """Whether torch has to see the call: to differentiate it, backwards or (which it refuses)
    forwards, or to record it in a trace."""
    if _tracing() is not None or (forward_ad._current_level >= 0 and _has_tangent(tensors)):
        return True
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors)


def _tensor(t, name: str, like=None, shape=None) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if like is not None:
        if t.device != like.device:
            raise RuntimeError(f"{name} must be on the same device as the other tensors")
        if t.dtype != like.dtype:
            raise RuntimeError(f"{name} must be {like.dtype}, the type of the other tensors")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")


def _stats(t, name: str, like, shape) -> torch.Tensor:
    """A float32 tensor of the forward pass, contiguous."""
    if not (isinstance(t, torch.Tensor) and t.device == like.device and t.dtype == torch.float32
            and tuple(t.shape) == tuple(shape)):
        raise RuntimeError(f"{name} must be a float32 tensor of shape {tuple(shape)} on the same device")
    return t.contiguous()


def _packed(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows(t: torch.Tensor, width: int, aligned: bool) -> torch.Tensor:
    """``t`` [..., width] as rows with unit column stride; ``aligned``: that start on 16 bytes."""
    r = t if t.dim() == 2 else t.reshape(-1, width)
    many = r.shape[0] > 1
    if r.stride(1) != 1 or (many and r.stride(0) < width):
        r = r.contiguous()
    if aligned and (r.data_ptr() % 16 != 0 or (many and (r.stride(0) % 8 != 0 or r.stride(0) > 1 << 21))):
        r = r.clone(memory_format=torch.contiguous_format)
    return r


def _row_stride(r: torch.Tensor) -> int:
    """The row stride; a single row's may be anything, and does not matter."""
    return r.stride(0) if r.shape[0] > 1 else r.shape[1]


def _workspace(key, like, plan):
    """Scratch of a call: its size by ``plan`` (asked once for each set of sizes)."""
    size = _plans.get(key)
    if size is None:
        out = _I64(0)
        _check(plan(ctypes.byref(out)))
        if len(_plans) >= 4096:
            _plans.clear()
        size = _plans[key] = int(out.value)
    return like.new_empty(size, dtype=torch.uint8) if size else None


def _new(t: torch.Tensor) -> torch.Tensor:
    """Contiguous memory for a result of t's shape and type."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- layer norm -----------------------------------------------------------------


def _norm_args(x, weight, bias):
    _tensor(x, "x")
    if x.dtype not in TYPES:
        raise RuntimeError("layer_norm takes float16, bfloat16 or float32")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError("x must be [..., width]")
    width = x.shape[-1]
    _tensor(weight, "weight", x, (width,))
    if bias is not None:
        _tensor(bias, "bias", x, (width,))
    return width


@_bare
def layer_norm_forward(x, weight, bias=None, eps: float = 1e-5, stats: bool = True):
    """(y, mean, rstd) of the rows of ``x`` [..., width]: y = (x - mean) rstd weight + bias
    with rstd = 1 / sqrt(variance + eps).  mean and rstd are float32 [...] for the
    backward pass, None without ``stats``."""
    width = _norm_args(x, weight, bias)
    lib = _library()
    r = _rows(x, width, False)
    y = _new(x)
    mean = rstd = None
    if stats:
        mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
        rstd = torch.empty_like(mean)
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    dev = x.device.index
    if r.shape[0]:
        _check(lib.cvs_layer_norm(r.data_ptr(), weight.data_ptr(), _ptr(bias), r.shape[0], width, _row_stride(r), eps,
                                  TYPES[x.dtype], y.data_ptr(), _ptr(mean), _ptr(rstd), dev, _ext.raw_stream(dev)))
    return y, mean, rstd


@_bare
def layer_norm_backward(dy, x, weight, mean, rstd):
    """(dx, dweight, dbias) of ``layer_norm_forward`` for ``dy``, of x's shape."""
    width = _norm_args(x, weight, None)
    _tensor(dy, "dy", x, x.shape)
    lib = _library()
    r, g = _rows(x, width, False), _rows(dy, width, False)
    n = r.shape[0]
    mean, rstd = _stats(mean, "mean", x, x.shape[:-1]), _stats(rstd, "rstd", x, x.shape[:-1])
    dx = _new(x)
    if n == 0:
        return dx, torch.zeros_like(weight), torch.zeros_like(weight)
    weight = weight.contiguous()
    dweight, dbias = torch.empty_like(weight), torch.empty_like(weight)
    dev, code = x.device.index, TYPES[x.dtype]
    ws = _workspace(("norm", n, width, code, dev), x,
                    lambda out: lib.cvs_layer_norm_backward_plan(n, width, code, dev, out))
    _check(lib.cvs_layer_norm_backward(g.data_ptr(), r.data_ptr(), weight.data_ptr(), mean.data_ptr(), rstd.data_ptr(), n,
                                       width, _row_stride(g), _row_stride(r), code, dx.data_ptr(), dweight.data_ptr(),
                                       dbias.data_ptr(), _ptr(ws), 0 if ws is None else ws.numel(), dev,
                                       _ext.raw_stream(dev)))
    return dx, dweight, dbias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward.inner(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.biased = bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx, dweight, dbias = layer_norm_backward.inner(dy, *ctx.saved_tensors)
        return dx, dweight, dbias if ctx.biased else None, None


def layer_norm(x, weight, bias=None, eps: float = 1e-5):
    """Layer norm over the last dimension of ``x``; ``weight`` and ``bias`` are [width]."""
    if _through_autograd(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_forward.inner(x, weight, bias, eps, stats=False)[0]


# ---- matrix product with its epilogue ----------------------------------------------


def _linear_args(x, weight, activation):
    _tensor(x, "x")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("linear takes float16 or bfloat16")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}")
    if x.dim() < 1:
        raise RuntimeError("x must be [..., in_features]")
    _tensor(weight, "weight", x)
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise RuntimeError("weight must be [out_features, in_features], as wide as x")
    n, k = weight.shape
    if k < 8 or n < 8 or k % 8 or n % 8:
        raise RuntimeError("linear takes feature counts that are multiples of 8 (zero-pad them)")
    return n, k


@_bare
def linear_forward(x, weight, bias=None, activation=None, residual=None, keep_pre: bool = False):
    """(y, pre): y = activation(x weight^T + bias) + residual for ``x`` [..., k] and ``weight``
    [n, k].  ``activation``: None, "gelu" (by the error function), "relu" or "tanh".
    pre is x weight^T + bias for the backward pass, None without ``keep_pre``."""
    n, k = _linear_args(x, weight, activation)
    shape = (*x.shape[:-1], n)
    if bias is not None:
        _tensor(bias, "bias", x, (n,))
    if residual is not None:
        _tensor(residual, "residual", x, shape)
    lib = _library()
    r = _rows(x, k, True)
    m = r.shape[0]
    y = x.new_empty(shape)
    pre = torch.empty_like(y) if keep_pre else None
    if m == 0:
        return y, pre
    weight = _packed(weight)
    bias = None if bias is None else _packed(bias)
    res = None if residual is None else _rows(residual, n, True)
    dev = x.device.index
    ws = _workspace(("linear", m, k, n, dev), x, lambda out: lib.cvs_linear_plan(m, k, n, dev, out))
    _check(lib.cvs_linear(r.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(res), m, k, n, _row_stride(r),
                          0 if res is None else _row_stride(res), ACTIVATIONS[activation], TYPES[x.dtype], y.data_ptr(),
                          _ptr(pre), _ptr(ws), 0 if ws is None else ws.numel(), dev, _ext.raw_stream(dev)))
    return y, pre


@_bare
def linear_backward(dy, x, weight, activation=None, pre=None, needs=(True, True, True)):
    """(dx, dweight, dbias) of ``linear_forward`` for ``dy``; the residual's gradient is ``dy``
    itself.  ``pre`` is what the forward pass kept (not needed without an
    activation).  Gradients that ``needs`` leaves out are None."""
    n, k = _linear_args(x, weight, activation)
    shape = (*x.shape[:-1], n)
    _tensor(dy, "dy", x, shape)
    if activation is not None:
        if pre is None:
            raise RuntimeError("pre, kept by the forward pass, is needed with an activation")
        _tensor(pre, "pre", x, shape)
        pre = _packed(pre)
    else:
        pre = None
    lib = _library()
    r, g = _rows(x, k, True), _rows(dy, n, True)
    m = r.shape[0]
    dx = _new(x) if needs[0] else None
    new = x.new_zeros if m == 0 else x.new_empty
    dweight = new((n, k)) if needs[1] else None
    dbias = new((n,)) if needs[2] else None
    if m == 0:
        return dx, dweight, dbias
    weight = _packed(weight)
    dev, act = x.device.index, ACTIVATIONS[activation]
    ws = _workspace(("linear backward", m, k, n, act, dev), x,
                    lambda out: lib.cvs_linear_backward_plan(m, k, n, act, dev, out))
    _check(lib.cvs_linear_backward(g.data_ptr(), r.data_ptr(), weight.data_ptr(), _ptr(pre), m, k, n, _row_stride(g),
                                   _row_stride(r), act, TYPES[x.dtype], _ptr(dx), _ptr(dweight), _ptr(dbias), _ptr(ws),
                                   0 if ws is None else ws.numel(), dev, _ext.raw_stream(dev)))
    return dx, dweight, dbias


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual):
        y, pre = linear_forward.inner(x, weight, bias, activation, residual, keep_pre=activation is not None)
        ctx.save_for_backward(x, weight, pre)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, pre = ctx.saved_tensors
        dx, dweight, dbias = linear_backward.inner(dy, x, weight, ctx.activation, pre, ctx.needs_input_grad[:3])
        return dx, dweight, dbias, None, dy if ctx.needs_input_grad[4] else None


def linear(x, weight, bias=None, activation=None, residual=None):
    """activation(x weight^T + bias) + residual; ``x`` [..., k], ``weight`` [n, k], feature
    counts multiples of 8."""
    if _through_autograd(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, activation, residual)
    return linear_forward.inner(x, weight, bias, activation, residual)[0]


# ---- attention -----------------------------------------------------------------------


def _lengths(t, name: str, q):
    if not (isinstance(t, torch.Tensor) and t.device == q.device and t.dtype == torch.int32
            and tuple(t.shape) == (q.shape[0],)):
        raise RuntimeError(f"{name} must be int32 [batch] on the same device")
    return t.contiguous()


def _strided(t: torch.Tensor):
    """(tensor, strides) of [batch, position, head, width] with rows of 16-byte pieces; a copy where it has none."""
    strides = [0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])]
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(s % 8 for s in strides) or strides[1] > 1 << 23:
        t = t.clone(memory_format=torch.contiguous_format)
        strides = list(t.stride()[:3])
    return t, _I64x3(*strides)


class _AttentionCall:
    """What a call's sizes, types and strides decide: checked, and filled in, once for all
    calls that have the same (checking each took 10 us of host time more)."""

    __slots__ = ("args", "bytes")

    def __init__(self, args):
        self.args = args
        self.bytes = [None, None]  # workspace of the forward and the backward pass


_calls: dict = {}


def _attention_check(q, k, v, bias_table, scale) -> None:
    _tensor(q, "q")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("attention takes float16 or bfloat16")
    _tensor(k, "k", q)
    _tensor(v, "v", q)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise RuntimeError("q must be [batch, q_len, heads, width], k and v [batch, k_len, k_heads, width]")
    width, heads = q.shape[3], q.shape[2]
    if k.shape[0] != q.shape[0] or k.shape[3] != width:
        raise RuntimeError("q, k and v must have the same batch and width")
    if width < 8 or width > 128 or width % 8:
        raise RuntimeError("attention takes head widths that are multiples of 8, at most 128")
    if heads < 1 or k.shape[2] < 1 or heads % k.shape[2]:
        raise RuntimeError("query heads must be a multiple of key heads")
    if bias_table is not None:
        _tensor(bias_table, "bias_table", q)
        if bias_table.dim() != 2 or bias_table.shape[1] != heads:
            raise RuntimeError("bias_table must be [buckets, heads]")


def _attention_args(q, k, v, bias_table, key_lengths, query_lengths, query_start, causal, scale, max_distance):
    """(AttentionArgs, its _AttentionCall or None, tensors it points into) after the checks."""
    # values, not tensors that hold them: those are found by identity and may have changed since
    scale = None if scale is None else float(scale)
    causal = bool(causal)
    max_distance = 0 if bias_table is None else operator.index(max_distance)
    try:
        key = (q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), q.dtype, k.dtype, v.dtype, q.device, k.device,
               v.device, causal, scale, max_distance,
               None if bias_table is None else (bias_table.shape, bias_table.dtype, bias_table.device))
        call = _calls.get(key)
    except (AttributeError, TypeError):  # no tensors: the checks say which
        key = call = None
    if call is None or (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        _attention_check(q, k, v, bias_table, scale)
        a = _ext.AttentionArgs()
        a.batch, a.q_len, a.heads, a.width = q.shape
        a.k_len, a.k_heads = k.shape[1:3]
        given = (q, k, v)
        q, a.q_stride = _strided(q)
        k, a.k_stride = _strided(k)
        v, a.v_stride = _strided(v)
        a.scale = 1.0 / math.sqrt(a.width) if scale is None else scale
        a.type, a.causal = TYPES[q.dtype], causal
        a.buckets, a.max_distance = (0, 0) if bias_table is None else (bias_table.shape[0], max_distance)
        call = None
        if key is not None and q is given[0] and k is given[1] and v is given[2]:
            if len(_calls) >= 4096:
                _calls.clear()
            call = _calls[key] = _AttentionCall(bytes(a))
    else:
        a = _ext.AttentionArgs.from_buffer_copy(call.args)
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    hold = [q, k, v]
    if bias_table is not None:
        bias_table = bias_table.contiguous()
        a.bias_table = bias_table.data_ptr()
        hold.append(bias_table)
    for name, lengths in (("key_lengths", key_lengths), ("query_lengths", query_lengths), ("query_start", query_start)):
        if lengths is not None:
            lengths = _lengths(lengths, name, q)
            setattr(a, name, lengths.data_ptr())
            hold.append(lengths)
    return a, call, hold


def _attention_workspace(lib, a, call, backward: bool, q):
    size = None if call is None else call.bytes[backward]
    if size is None:
        out = _I64(0)
        _check(lib.cvs_attention_plan(ctypes.byref(a), backward, q.device.index, ctypes.byref(out)))
        size = int(out.value)
        if call is not None:
            call.bytes[backward] = size
    return q.new_empty(size, dtype=torch.uint8) if size else None


@_bare
def attention_forward(q, k, v, bias_table=None, key_lengths=None, query_lengths=None, query_start=None,
                      causal: bool = False, scale=None, max_distance: int = 128, lse: bool = True):
    """(out, lse) of softmax attention: ``q`` [batch, q_len, heads, width], ``k`` and ``v``
    [batch, k_len, k_heads, width] (any strides whose rows of ``width`` are contiguous), out like q,
    lse float32 [batch, heads, q_len] (natural logarithm; None when not asked for).

    Query head h reads key head h // (heads // k_heads).  Row i of sequence b stands at key
    position i + start, start = ``query_start[b]`` (by default k_len - q_len: the last row at the
    last key), and sees key j when j < ``key_lengths[b]`` and, if ``causal``, j <= i + start.
    Rows at or past ``query_lengths[b]`` see nothing; a row that sees nothing has out 0 and
    lse -inf.  What lies in keys that no row sees (a cache's places not yet written)
    reaches no result.  ``scale`` is from 2^-100 to 2^100, by default width ** -0.5.

    ``bias_table`` [buckets, heads] adds bias_table[bucket(j - i - start), h] to the score.
    Buckets: half of a direction's for one distance each, the others evenly in the
    logarithm up to ``max_distance`` (the last one also holds what is further); causal: all
    buckets for the past, else the first half for keys at or before the row.
    """
    a, call, hold = _attention_args(q, k, v, bias_table, key_lengths, query_lengths, query_start, causal, scale, max_distance)
    lib = _library()
    out = _new(q)
    sums = q.new_empty((a.batch, a.heads, a.q_len), dtype=torch.float32) if lse else None
    dev = q.device.index
    ws = _attention_workspace(lib, a, call, False, q)
    _check(lib.cvs_attention_forward(ctypes.byref(a), out.data_ptr(), _ptr(sums), _ptr(ws), 0 if ws is None else ws.numel(),
                                     dev, _ext.raw_stream(dev)))
    return out, sums


@_bare
def attention_backward(dout, q, k, v, out, lse, bias_table=None, key_lengths=None, query_lengths=None, query_start=None,
                       causal: bool = False, scale=None, max_distance: int = 128):
    """(dq, dk, dv, dbias_table) of ``attention_forward`` for ``dout``, from its ``out`` and ``lse``;
    dbias_table is None without a table."""
    a, call, hold = _attention_args(q, k, v, bias_table, key_lengths, query_lengths, query_start, causal, scale, max_distance)
    _tensor(dout, "dout", q, q.shape)
    _tensor(out, "out", q, q.shape)
    lse = _stats(lse, "lse", q, (a.batch, a.heads, a.q_len))
    lib = _library()
    dout, dout_stride = _strided(dout)
    out = _packed(out)
    dq, dk, dv = _new(q), _new(k), _new(v)
    dtable = None if bias_table is None else torch.empty_like(hold[3])
    if a.batch == 0 or (a.q_len == 0 and a.k_len == 0):
        return dq, dk, dv, None if dtable is None else dtable.zero_()
    dev = q.device.index
    ws = _attention_workspace(lib, a, call, True, q)
    _check(lib.cvs_attention_backward(ctypes.byref(a), dout.data_ptr(), dout_stride, out.data_ptr(), lse.data_ptr(),
                                      dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dtable), _ptr(ws),
                                      0 if ws is None else ws.numel(), dev, _ext.raw_stream(dev)))
    return dq, dk, dv, dtable


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias_table, key_lengths, query_lengths, query_start, causal, scale, max_distance):
        out, lse = attention_forward.inner(q, k, v, bias_table, key_lengths, query_lengths, query_start, causal, scale, max_distance)
        ctx.save_for_backward(q, k, v, out, lse, bias_table, key_lengths, query_lengths, query_start)
        ctx.more = (causal, scale, max_distance)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, *masks = ctx.saved_tensors
        return (*attention_backward.inner(dout, q, k, v, out, lse, *masks, *ctx.more), None, None, None, None, None, None)


def attention(q, k, v, bias_table=None, key_lengths=None, query_lengths=None, query_start=None, causal: bool = False,
              scale=None, max_distance: int = 128):
    """Softmax attention, [batch, q_len, heads, width]; arguments as ``attention_forward``'s."""
    args = (q, k, v, bias_table, key_lengths, query_lengths, query_start, causal, scale, max_distance)
    if _through_autograd(q, k, v, bias_table):
        return _Attention.apply(*args)
    return attention_forward.inner(*args, lse=False)[0]
