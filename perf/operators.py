"""Performance cases of the text-encoder operators, with their plain forms.

Each case is a plain dict.  ``op`` and ``pass`` name the call that is timed:

* ``"norm"``   - ``layer_norm_forward`` / ``layer_norm_backward`` of ``rows`` x ``width``;
* ``"linear"`` - ``linear_forward`` / ``linear_backward`` of ``rows`` tokens, ``k`` to ``n``
  features, with bias, ``act`` and (``residual``) a residual; ``keep``: the forward pass
  also returns the values before the activation, as training needs them;
* ``"attn"``   - ``attention_forward`` / ``attention_backward`` of ``b`` sequences of ``lq`` queries
  and ``lk`` keys, ``h`` query heads, ``hk`` key heads of width ``d``; ``buckets`` > 0: a learned
  bias by relative position; ``ragged``: the sequences' lengths vary; ``causal``.

``dtype`` is that of the inputs; results have it too (row statistics are float32).
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-5
_MAX_DISTANCE = 128

_LISTED = [
    # The norm of one short query: all latency.
    {"name": "norm_query", "op": "norm", "pass": "forward", "dtype": "fp16", "rows": 23, "width": 384},
    # A training batch of 128 passages of 128 tokens.
    {"name": "norm_train_bwd", "op": "norm", "pass": "backward", "dtype": "bf16", "rows": 16384, "width": 768},
    # Parameters and activations kept in 32 bits, a row count and width that are multiples of little.
    {"name": "norm_fp32_bwd", "op": "norm", "pass": "backward", "dtype": "fp32", "rows": 50021, "width": 1000},
    # The first feed-forward product of one short query: the weights are what is read.
    {"name": "linear_query", "op": "linear", "pass": "forward", "dtype": "fp16", "rows": 23, "k": 384, "n": 1536,
     "act": "gelu", "residual": False, "keep": False},
    # The same product in training, wide rows: keeps what the backward pass needs.
    {"name": "linear_up_train", "op": "linear", "pass": "forward", "dtype": "bf16", "rows": 16384, "k": 768, "n": 2048,
     "act": "gelu", "residual": False, "keep": True},
    # The second product over a ragged batch of passages, with the residual.
    {"name": "linear_down", "op": "linear", "pass": "forward", "dtype": "fp16", "rows": 10007, "k": 2048, "n": 768,
     "act": "none", "residual": True, "keep": False},
    # Gradients of the first feed-forward product.
    {"name": "linear_up_bwd", "op": "linear", "pass": "backward", "dtype": "bf16", "rows": 16384, "k": 768, "n": 2048,
     "act": "gelu", "residual": False, "keep": False},
    # Self-attention of one short query.
    {"name": "attn_query", "op": "attn", "pass": "forward", "dtype": "fp16", "b": 1, "lq": 23, "lk": 23, "h": 12, "hk": 12,
     "d": 32, "buckets": 32, "ragged": False, "causal": False},
    # One pooling token a document over all its tokens.
    {"name": "attn_pool", "op": "attn", "pass": "forward", "dtype": "fp16", "b": 8, "lq": 1, "lk": 8191, "h": 12, "hk": 12,
     "d": 64, "buckets": 0, "ragged": True, "causal": False},
    # Passages being embedded: sequences of up to 512 tokens.
    {"name": "attn_passages", "op": "attn", "pass": "forward", "dtype": "fp16", "b": 64, "lq": 512, "lk": 512, "h": 12, "hk": 12,
     "d": 64, "buckets": 32, "ragged": True, "causal": False},
    # A training batch of passages: gradients, the bias table's among them.
    {"name": "attn_train_bwd", "op": "attn", "pass": "backward", "dtype": "bf16", "b": 32, "lq": 512, "lk": 512, "h": 12,
     "hk": 12, "d": 64, "buckets": 32, "ragged": True, "causal": False},
    # Long documents, a causal encoder with shared key heads.
    {"name": "attn_long_bwd", "op": "attn", "pass": "backward", "dtype": "bf16", "b": 2, "lq": 4096, "lk": 4096, "h": 16, "hk": 4,
     "d": 128, "buckets": 0, "ragged": False, "causal": True},
]


def listed():
    return [dict(c) for c in _LISTED]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    """A rough time (s) of an ordinary implementation."""
    w = work(case)
    return w["bytes"] / 3e12 + w["flops"] / 4e14


def _widths(rng, hi):
    """Feature counts: common ones, and one in three any multiple of 8."""
    if rng.random() < 0.34:
        return 8 * _log_int(rng, 8, hi // 8)
    return rng.choice([w for w in (64, 128, 256, 384, 512, 768, 1024, 1536, 2048) if w <= hi])


def draw(rng):
    """One more case of the same ranges: rows from 1 to 50k, widths to 2048, sequences
    from 1 token to 8k, both directions, all types."""
    most = max(_cost(c) for c in _LISTED)
    while True:
        op = rng.choice(["norm", "linear", "attn"])
        case = {"op": op, "pass": rng.choice(["forward", "backward"]), "dtype": rng.choice(["fp16", "bf16"])}
        if op == "norm":
            case["dtype"] = rng.choice(["fp16", "bf16", "fp32"])
            case["rows"] = _log_int(rng, 1, 50_000)
            case["width"] = _widths(rng, 2048) if rng.random() < 0.7 else _log_int(rng, 33, 2048)
        elif op == "linear":
            case["rows"] = _log_int(rng, 1, 30_000)
            case["k"], case["n"] = _widths(rng, 2048), _widths(rng, 2048)
            case["act"] = rng.choice(["none", "gelu", "gelu", "relu", "tanh"])
            case["residual"] = case["pass"] == "forward" and rng.random() < 0.4
            case["keep"] = case["pass"] == "forward" and case["act"] != "none" and rng.random() < 0.5
        else:
            case["b"] = _log_int(rng, 1, 64)
            case["lk"] = _log_int(rng, 1, 8192)
            case["lq"] = case["lk"] if rng.random() < 0.75 else 1 if rng.random() < 0.5 else _log_int(rng, 1, case["lk"])
            case["hk"] = rng.choice([1, 2, 4, 12])
            case["h"] = case["hk"] * rng.choice([1, 1, 2, 4])
            case["d"] = rng.choice([32, 64, 64, 128, 8 * rng.randint(3, 16)])
            case["buckets"] = rng.choice([0, 32, 32, 64])
            case["ragged"] = rng.random() < 0.5
            case["causal"] = rng.random() < 0.35
            if case["b"] * case["h"] * case["lq"] * case["lk"] > 1 << 29:
                continue
        if _cost(case) <= most:
            return case


# ---- inputs -----------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 31)


def _hidden(shape, g, dtype):
    """Hidden states: channels of different spread and offset, a few of them large."""
    width = shape[-1]
    spread = torch.exp(0.4 * torch.randn(width, device="cuda", generator=g))
    shift = 0.2 * torch.randn(width, device="cuda", generator=g)
    return (torch.randn(*shape, device="cuda", generator=g) * spread + shift).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    dtype = _DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0):
        return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)

    s = {"case": dict(case)}
    back = case["pass"] == "backward"
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        s["x"] = _hidden((rows, width), g, dtype)
        s["weight"] = (1.0 + 0.2 * torch.randn(width, device="cuda", generator=g)).to(dtype)
        s["bias"] = rand(width, scale=0.1)
        if back:  # the forward pass's statistics are in hand
            xf = s["x"].float()
            s["mean"] = xf.mean(1)
            s["rstd"] = ((xf - s["mean"][:, None]).square().mean(1) + _EPS).rsqrt()
            s["dy"] = rand(rows, width, scale=0.5)
    elif case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"] = _hidden((rows, k), g, dtype)
        s["weight"] = rand(n, k, scale=1.0 / math.sqrt(k))
        s["bias"] = rand(n, scale=0.2)
        s["residual"] = rand(rows, n) if case["residual"] and not back else None
        if back:
            s["dy"] = rand(rows, n, scale=0.5)
            s["pre"] = rand(rows, n, scale=1.2) if case["act"] != "none" else None
    else:
        b, lq, lk, h, hk, d = (case[c] for c in ("b", "lq", "lk", "h", "hk", "d"))
        if lq == lk and h == hk:  # one projection's output, split
            qkv = rand(b, lq, 3, h, d)
            qkv[:, :, 0] *= 1.5
            s["q"], s["k"], s["v"] = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
        else:
            s["q"], s["k"], s["v"] = rand(b, lq, h, d, scale=1.5), rand(b, lk, hk, d), rand(b, lk, hk, d)
        s["table"] = rand(case["buckets"], h) if case["buckets"] else None
        s["key_lengths"] = s["query_lengths"] = None
        if case["ragged"]:  # between a quarter of the longest and all of it
            u = torch.rand(b, device="cuda", generator=g)
            s["key_lengths"] = ((0.25 + 0.75 * u) * lk).ceil().clamp(1, lk).to(torch.int32)
            if lq == lk:
                s["query_lengths"] = s["key_lengths"]
        if back:  # the forward pass's results are in hand
            s["out"], s["lse"] = _attention_forward(s)
            s["dout"] = rand(b, lq, h, d, scale=0.5)
    return s


# ---- plain forms, in 32 bits --------------------------------------------------


def _norm_forward(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = ((xc * xc).mean(1, keepdim=True) + _EPS).rsqrt()
    y = xc * rstd * s["weight"].float() + s["bias"].float()
    return y.to(s["x"].dtype), mean[:, 0], rstd[:, 0]


def _norm_backward(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["weight"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    t = s["x"].dtype
    return dx.to(t), (dy * xhat).sum(0).to(t), dy.sum(0).to(t)


def _activate(z, act):
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    return torch.tanh(z) if act == "tanh" else z


def _slope(z, act):
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "relu":
        return (z > 0).to(z.dtype)
    return 1.0 - torch.tanh(z).square()


def _linear_forward(s):
    z = s["x"].float() @ s["weight"].float().T + s["bias"].float()
    y = _activate(z, s["case"]["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    t = s["x"].dtype
    return (y.to(t), z.to(t)) if s["case"]["keep"] else (y.to(t),)


def _linear_backward(s):
    dz = s["dy"].float()
    if s["pre"] is not None:
        dz = dz * _slope(s["pre"].float(), s["case"]["act"])
    t = s["x"].dtype
    return (dz @ s["weight"].float()).to(t), (dz.T @ s["x"].float()).to(t), dz.sum(0).to(t)


def _boundaries(buckets, causal):
    """Smallest distances of the buckets past the first half (those hold one distance each)."""
    one_way = buckets if causal else buckets // 2
    exact = one_way // 2
    wide = one_way - exact
    return exact, one_way, [math.ceil(exact * (_MAX_DISTANCE / exact) ** (t / wide) - 1e-9) for t in range(1, wide)]


def _bucket(rel, buckets, causal):
    """Bucket of the relative positions ``rel`` = key - query: the sign's half (none where only
    the past is seen), one bucket a distance for the nearest, then evenly in the logarithm."""
    exact, one_way, bounds = _boundaries(buckets, causal)
    dist = (-rel).clamp(min=0) if causal else rel.abs()
    far = exact + torch.searchsorted(torch.tensor(bounds, device=rel.device), dist, right=True)
    found = torch.where(dist < exact, dist, far)
    return found if causal else found + one_way * (rel > 0)


def _positions(c, device):
    """Key minus query positions; the last query stands at the last key."""
    i = torch.arange(c["lq"], device=device) + (c["lk"] - c["lq"])
    return torch.arange(c["lk"], device=device)[None, :] - i[:, None]


def _heads(t):
    return t.transpose(1, 2)


def _attention_parts(s):
    """(q, k, v [b, h, l, d], probabilities, log sums, row mask or None, buckets or None) in 32 bits."""
    c = s["case"]
    dev = s["q"].device
    group = c["h"] // c["hk"]
    q, k, v = (_heads(s[n]).float() for n in ("q", "k", "v"))
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    scores = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(c["d"]))
    rel, found = _positions(c, dev), None
    if s["table"] is not None:
        found = _bucket(rel, c["buckets"], c["causal"])
        scores = scores + s["table"].float()[found].permute(2, 0, 1)
    if c["causal"]:
        scores = scores.masked_fill(rel > 0, -math.inf)
    if s["key_lengths"] is not None:
        past = torch.arange(c["lk"], device=dev) >= s["key_lengths"][:, None]
        scores = scores.masked_fill(past[:, None, None, :], -math.inf)
    rows = None
    if s["query_lengths"] is not None:
        rows = (torch.arange(c["lq"], device=dev) >= s["query_lengths"][:, None])[:, None, :, None]
        scores = scores.masked_fill(rows, -math.inf)
    top = scores.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(scores - top)
    total = e.sum(3, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    return q, k, v, p, (top + torch.log(total))[..., 0], rows, found


def _attention_forward(s):
    _, _, v, p, lse, _, _ = _attention_parts(s)
    return _heads(p @ v).contiguous().to(s["q"].dtype), lse


def _shared(t, c):
    """Sum over the query heads of each key head."""
    return t.reshape(c["b"], c["hk"], c["h"] // c["hk"], c["lk"], c["d"]).sum(2)


def _attention_backward(s):
    c, t = s["case"], s["q"].dtype
    q, k, v, p, _, _, found = _attention_parts(s)
    do = _heads(s["dout"]).float()
    scale = 1.0 / math.sqrt(c["d"])
    dv = _shared(p.transpose(2, 3) @ do, c)
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    dq = (ds @ k) * scale
    dk = _shared(ds.transpose(2, 3) @ q, c) * scale
    grads = [_heads(x).contiguous().to(t) for x in (dq, dk, dv)]
    if found is not None:
        by_pair = ds.sum(0).reshape(c["h"], -1).T
        grads.append(torch.zeros(c["buckets"], c["h"], device=q.device).index_add_(0, found.reshape(-1), by_pair).to(t))
    return tuple(grads)


_PLAIN = {("norm", "forward"): _norm_forward, ("norm", "backward"): _norm_backward,
          ("linear", "forward"): _linear_forward, ("linear", "backward"): _linear_backward,
          ("attn", "forward"): _attention_forward, ("attn", "backward"): _attention_backward}


# ---- the framework's calls ------------------------------------------------------


def _package():
    root = str(Path(__file__).resolve().parents[1] / "cuda-vector-search_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from cuda_vector_search import encoder

    return encoder


def run(s):
    c = s["case"]
    if not own:
        return _PLAIN[c["op"], c["pass"]](s)
    e = _package()
    back = c["pass"] == "backward"
    if c["op"] == "norm":
        if back:
            return e.layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"])
        return e.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=_EPS)
    if c["op"] == "linear":
        act = None if c["act"] == "none" else c["act"]
        if back:
            return e.linear_backward(s["dy"], s["x"], s["weight"], activation=act, pre=s["pre"])
        y, pre = e.linear_forward(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"],
                                  keep_pre=c["keep"])
        return (y, pre) if c["keep"] else (y,)
    more = {"bias_table": s["table"], "key_lengths": s["key_lengths"], "query_lengths": s["query_lengths"],
            "causal": c["causal"], "max_distance": _MAX_DISTANCE}
    if not back:
        return e.attention_forward(s["q"], s["k"], s["v"], **more)
    grads = e.attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], **more)
    return grads if s["table"] is not None else grads[:3]


# ---- what a pass cannot do without ------------------------------------------------


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    back = case["pass"] == "backward"
    if case["op"] == "norm":
        cells = case["rows"] * case["width"]
        return {"bytes": size * (3 if back else 2) * cells + 8 * case["rows"] + 3 * size * case["width"],
                "flops": (12 if back else 8) * cells}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        if back:
            wide = 1 if case["act"] == "none" else 2
            return {"bytes": size * (wide * m * n + 2 * m * k + 2 * n * k + n), "flops": 4 * m * n * k}
        wide = 1 + bool(case["residual"]) + bool(case["keep"])
        return {"bytes": size * (m * k + n * k + wide * m * n + n), "flops": 2 * m * n * k}
    b, lq, lk, h, hk, d = (case[c] for c in ("b", "lq", "lk", "h", "hk", "d"))
    pairs, q_rows, k_rows = float(lq * lk), float(lq), float(lk)
    if case["causal"]:
        pairs = lq * (lk - lq) + lq * (lq + 1) / 2
    if case["ragged"]:  # mean lengths: 5/8 of the longest; the mean of their squares: 7/16
        pairs *= 7 / 16 if lq == lk else 5 / 8
        k_rows *= 5 / 8
        q_rows *= 5 / 8 if lq == lk else 1
    rows_q, rows_k = b * h * q_rows * d, b * hk * k_rows * d
    if back:  # q, out, dout in, dq out; k, v in, dk, dv out; the log sums
        return {"bytes": size * (4 * rows_q + 4 * rows_k) + 4 * b * h * q_rows, "flops": 10 * b * h * pairs * d}
    return {"bytes": size * (2 * rows_q + 2 * rows_k) + 4 * b * h * q_rows, "flops": 4 * b * h * pairs * d}


# ---- the definitions, in 64 bits ---------------------------------------------------


def _exact_norm(c, s):
    x, w = s["x"].double(), s["weight"].double()
    n = c["width"]
    mu = x.sum(1, keepdim=True) / n
    dev = torch.sqrt(((x - mu) ** 2).sum(1, keepdim=True) / n + _EPS)
    unit = (x - mu) / dev
    if c["pass"] == "forward":
        return unit * w + s["bias"].double(), mu.squeeze(1), 1.0 / dev.squeeze(1)
    dy = s["dy"].double()
    # y = unit * w + b: the Jacobian of unit is (I - 1/n - unit unit^T / n) / dev
    u = dy * w
    dx = (u - u.sum(1, keepdim=True) / n - unit * ((u * unit).sum(1, keepdim=True) / n)) / dev
    return dx, torch.einsum("rc,rc->c", dy, unit), dy.sum(0)


def _exact_linear(c, s):
    x, w = s["x"].double(), s["weight"].double()
    normal = torch.distributions.Normal(torch.zeros((), device="cuda", dtype=torch.float64),
                                        torch.ones((), device="cuda", dtype=torch.float64))
    if c["pass"] == "forward":
        z = torch.addmm(s["bias"].double(), x, w.t())
        y = {"gelu": lambda: z * normal.cdf(z), "relu": lambda: z.clamp(min=0), "tanh": lambda: z.tanh(),
             "none": lambda: z}[c["act"]]()
        if s["residual"] is not None:
            y = y + s["residual"].double()
        return (y, z) if c["keep"] else (y,)
    g = s["dy"].double()
    if s["pre"] is not None:
        z = s["pre"].double()
        g = g * {"gelu": lambda: normal.cdf(z) + z * normal.log_prob(z).exp(), "relu": lambda: z.gt(0).double(),
                 "tanh": lambda: z.cosh() ** -2}[c["act"]]()
    return torch.mm(g, w), torch.mm(g.t().contiguous(), x), g.sum(0)


def _exact_attention(c, s):
    """One sequence and key head at a time."""
    b, lq, lk, h, hk, d = (c[n] for n in ("b", "lq", "lk", "h", "hk", "d"))
    group, back, dev = h // hk, c["pass"] == "backward", "cuda"
    f64 = {"dtype": torch.float64, "device": dev}
    out, lse = torch.zeros(b, lq, h, d, **f64), torch.full((b, h, lq), -math.inf, **f64)
    dq, dk, dv = torch.zeros(b, lq, h, d, **f64), torch.zeros(b, lk, hk, d, **f64), torch.zeros(b, lk, hk, d, **f64)
    # bucket of each distance, by counting: a boundary at exact * (max / exact)^(t / wide)
    bias_of = dtable = None
    rel = torch.arange(lk, device=dev).unsqueeze(0) - torch.arange(lq, device=dev).unsqueeze(1) - (lk - lq)
    if c["buckets"]:
        one = c["buckets"] if c["causal"] else c["buckets"] // 2
        exact = one // 2
        steps = torch.arange(1, one - exact, **f64)
        edges = torch.ceil(exact * torch.pow(torch.tensor(_MAX_DISTANCE / exact, **f64), steps / (one - exact)) - 1e-9)
        far = torch.arange(lk + lq + 1, **f64)
        by_distance = torch.minimum(far, torch.full_like(far, exact)) + (far[:, None] >= edges).sum(1) * (far >= exact)
        ahead = 0 if c["causal"] else one
        length = (-rel).clamp(min=0) if c["causal"] else rel.abs()
        bias_of = by_distance.long()[length] + ahead * (rel > 0).long()
        dtable = torch.zeros(c["buckets"], h, **f64)
        pair_sum = torch.zeros(h, lq, lk, **f64)
    klen = [lk] * b if s["key_lengths"] is None else s["key_lengths"].tolist()
    qlen = [lq] * b if s["query_lengths"] is None else s["query_lengths"].tolist()
    for n in range(b):
        nq, nk = qlen[n], klen[n]
        if not nq or not nk:
            continue
        r = rel[:nq, :nk]
        for head in range(h):
            kv = head // group
            q, k, v = s["q"][n, :nq, head].double(), s["k"][n, :nk, kv].double(), s["v"][n, :nk, kv].double()
            z = torch.mm(q, k.t()) / math.sqrt(d)
            if bias_of is not None:
                z = z + s["table"][:, head].double()[bias_of[:nq, :nk]]
            if c["causal"]:
                z = torch.where(r > 0, torch.full_like(z, -math.inf), z)
            total = torch.logsumexp(z, 1)
            p = torch.exp(z - torch.where(total == -math.inf, torch.zeros_like(total), total)[:, None])
            if not back:
                out[n, :nq, head], lse[n, head, :nq] = torch.mm(p, v), total
                continue
            do = s["dout"][n, :nq, head].double()
            dv[n, :nk, kv] += torch.mm(p.t(), do)
            dp = torch.mm(do, v.t())
            dz = p * dp - p * (p * dp).sum(1, keepdim=True)
            dq[n, :nq, head] = torch.mm(dz, k) / math.sqrt(d)
            dk[n, :nk, kv] += torch.mm(dz.t(), q) / math.sqrt(d)
            if bias_of is not None:
                pair_sum[head, :nq, :nk] += dz
    if not back:
        return out, lse
    if dtable is None:
        return dq, dk, dv
    for head in range(h):
        dtable[:, head] = torch.bincount(bias_of.reshape(-1), pair_sum[head].reshape(-1), c["buckets"])
    return dq, dk, dv, dtable


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "linear": _exact_linear, "attn": _exact_attention}[case["op"]](case, s)
