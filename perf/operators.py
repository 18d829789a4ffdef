"""What the text-encoder operators are measured on: cases, plain forms, exact values.

Three operators of `coda_wan_dit_b200.ops`, the parts of a text encoder's layer whose output the
diffusion transformer's cross-attention reads:

* ``rel_pos_bias`` / ``rel_pos_bias_grad``: a learned relative position bias by buckets;
* ``rel_pos_attention``: attention that reads that bias from its table;
* ``linear_act_residual``: act(x W^T + b) + r.

``own`` false computes the plain form (elementary torch operations in 32 bits, rounded once),
true calls the framework.
"""
from __future__ import annotations

import math
from functools import lru_cache

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _ops():
    from __graft_entry__ import load_package

    return load_package().ops


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _bias(name, heads, q_len, k_len, dtype, q_offset=0, buckets=32, max_distance=128, bidirectional=True):
    return dict(name=name, kind="bias", heads=heads, q_len=q_len, k_len=k_len, q_offset=q_offset, buckets=buckets,
                max_distance=max_distance, bidirectional=bidirectional, dtype=dtype)


def _bias_grad(name, batch, heads, q_len, k_len, dtype, q_offset=0, buckets=32, max_distance=128,
               bidirectional=True):
    c = _bias(name, heads, q_len, k_len, dtype, q_offset, buckets, max_distance, bidirectional)
    c.update(kind="bias_grad", batch=batch)
    return c


def _linear(name, m, n, k, dtype, act, bias=True, residual=True, train=False):
    return dict(name=name, kind="linear_train" if train else "linear", m=m, n=n, k=k, dtype=dtype, act=act,
                bias=bias, residual=residual)


def _attn(name, batch, heads, head_dim, q_len, k_len, dtype, len_step=0, q_offset=0, causal=False,
          bidirectional=True, buckets=32, max_distance=128, unit_scale=False, train=False):
    # sample b has max(0, k_len - b * len_step) valid keys (prompts padded to one length)
    return dict(name=name, kind="attn_train" if train else "attn", batch=batch, heads=heads, head_dim=head_dim,
                q_len=q_len, k_len=k_len, len_step=len_step, q_offset=q_offset, causal=causal,
                bidirectional=bidirectional, buckets=buckets, max_distance=max_distance, unit_scale=unit_scale,
                dtype=dtype)


def listed():
    return [
        # one layer's bias for a prompt padded to the text length (512), 64 heads
        _bias("bias_text", 64, 512, 512, "bf16"),
        # the bias row of one generated token over its cache: latency
        _bias("bias_token", 12, 1, 4097, "fp32", q_offset=4096, bidirectional=False),
        # its gradient from a fine-tuning step's score gradients, two prompts
        _bias_grad("bias_grad_text", 2, 64, 512, 512, "bf16"),
        # ... over long odd lengths, one head group, 32-bit scores
        _bias_grad("bias_grad_long", 1, 40, 2047, 2049, "fp32", buckets=64, max_distance=500),
        # one token through a feed-forward layer's second product: reads the weight once
        _linear("linear_token", 1, 1536, 8960, "bf16", "none"),
        # two padded prompts into the model width (the text projection), tanh-GELU, no residual
        _linear("linear_text", 1024, 1536, 4096, "bf16", "gelu_tanh", residual=False),
        # a wide feed-forward layer over a long batch, half precision
        _linear("linear_wide", 8192, 13824, 5120, "fp16", "gelu"),
        # a fine-tuning step of the feed-forward's first product, ragged token count
        _linear("linear_train", 4095, 8960, 1536, "bf16", "silu", train=True),
        # encoder self-attention over two padded prompts, unscaled scores
        _attn("attn_text", 2, 64, 64, 512, 512, "bf16", len_step=285, unit_scale=True),
        # one generated token a sequence over long caches of different lengths
        _attn("attn_token", 8, 12, 128, 1, 8191, "fp16", len_step=700, q_offset=8190, causal=False,
              bidirectional=False),
        # a long document, causal
        _attn("attn_long", 1, 12, 128, 8192, 8192, "bf16", causal=True, bidirectional=False),
        # a fine-tuning step of the encoder's attention, gradients of q, k, v and the table
        _attn("attn_train", 2, 64, 64, 512, 512, "bf16", len_step=131, unit_scale=True, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    kind = rng.choice(["bias", "bias_grad", "linear", "linear", "linear_train", "attn", "attn", "attn_train"])
    buckets, max_distance = rng.choice([(32, 128), (32, 128), (16, 100), (64, 500), (32, 1000)])
    bidirectional = rng.random() < 0.6
    pos = dict(buckets=buckets, max_distance=max_distance, bidirectional=bidirectional)
    half = rng.choice(["bf16", "fp16"])
    if kind in ("bias", "bias_grad"):
        heads = _log_int(rng, 1, 64)
        q_len = _log_int(rng, 1, 2048)
        k_len = _log_int(rng, 1, 4096)
        while heads * q_len * k_len > 64 << 20:
            heads = max(1, heads // 2)
        off = 0 if bidirectional and rng.random() < 0.7 else max(0, k_len - q_len)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        if kind == "bias":
            return _bias(None, heads, q_len, k_len, dtype, off, **pos)
        return _bias_grad(None, rng.choice([1, 1, 2, 3]), heads, q_len, k_len, dtype, off, **pos)
    if kind in ("linear", "linear_train"):
        act = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"])
        n = 8 * _log_int(rng, 8, 1728)
        k = 8 * _log_int(rng, 8, 1728)
        train = kind == "linear_train"
        m = _log_int(rng, 1, 8192)
        while m * n * k * (3 if train else 1) > 3 << 37:
            m = max(1, m // 2)
        return _linear(None, m, n, k, half, act, rng.random() < 0.8, rng.random() < 0.6, train)
    head_dim = rng.choice([64, 128])
    batch = rng.choice([1, 2, 3, 5])
    heads = _log_int(rng, 1, 64)
    if kind == "attn" and rng.random() < 0.5:  # tokens after a cache
        q_len = rng.choice([1, 1, 1, 2, 5, 16])
        k_len = _log_int(rng, max(q_len, 8), 16384)
        while batch * heads * k_len * head_dim > 1 << 27:
            heads = max(1, heads // 2)
        step = rng.choice([0, k_len // 7, k_len // 2])
        return _attn(None, batch, heads, head_dim, q_len, k_len, half, step, k_len - q_len, rng.random() < 0.5,
                     rng.random() < 0.3, buckets, max_distance, False, False)
    q_len = _log_int(rng, 1, 4096)
    causal = rng.random() < 0.4
    k_len = q_len if rng.random() < 0.7 else _log_int(rng, 1, 4096)
    while batch * heads * q_len * k_len > 1 << 28:
        heads, batch = (max(1, heads // 2), batch) if heads > 1 else (1, 1)
        if heads == 1 and batch == 1:
            break
    step = rng.choice([0, k_len // 5, k_len // 3, k_len])
    return _attn(None, batch, heads, head_dim, q_len, k_len, half, step, max(0, k_len - q_len) if causal else 0,
                 causal, bidirectional and not causal, buckets, max_distance, rng.random() < 0.5,
                 kind == "attn_train")


# ---------------------------------------------------------------------------
# The bucket of a relative position
# ---------------------------------------------------------------------------
@lru_cache(maxsize=None)
def _bounds(buckets, max_distance, bidirectional):
    """Ascending distances at which the bucket steps up by one: the bucket of distance n is the
    number of bounds <= n. Distances below `exact` have a bucket each; bucket exact + t begins at
    the least n with n^T >= max_distance^t exact^(T - t) (the logarithmic rule in whole numbers)."""
    nb = buckets // 2 if bidirectional else buckets
    exact = nb // 2
    T = nb - exact
    out = list(range(1, exact + 1))
    for t in range(1, T):
        target = max_distance**t * exact ** (T - t)
        lo, hi = exact, max_distance
        while lo < hi:
            mid = (lo + hi) // 2
            if mid**T >= target:
                hi = mid
            else:
                lo = mid + 1
        out.append(lo)
    return tuple(out)


def _buckets(case, device, q_lo=0, q_hi=None):
    """[q_hi - q_lo, k_len] bucket numbers of key j seen from query i + q_offset."""
    q_hi = case["q_len"] if q_hi is None else q_hi
    i = torch.arange(q_lo, q_hi, device=device)[:, None] + case["q_offset"]
    d = torch.arange(case["k_len"], device=device)[None, :] - i
    bounds = torch.tensor(_bounds(case["buckets"], case["max_distance"], case["bidirectional"]), device=device)
    n = d.abs() if case["bidirectional"] else (-d).clamp_min(0)
    b = torch.searchsorted(bounds, n, right=True)
    if case["bidirectional"]:
        b = b + (d > 0) * (case["buckets"] // 2)
    return b


def _lens(case):
    return [max(0, case["k_len"] - b * case["len_step"]) for b in range(case["batch"])]


def _scale(case):
    return 1.0 if case["unit_scale"] else case["head_dim"] ** -0.5


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def randn(*shape, dtype=dt, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)

    s = {"case": case}
    kind = case["kind"]
    if kind == "bias":
        s["table"] = randn(case["buckets"], case["heads"])
    elif kind == "bias_grad":
        s["dbias"] = randn(case["batch"], case["heads"], case["q_len"], case["k_len"])
    elif kind in ("linear", "linear_train"):
        m, n, k = case["m"], case["n"], case["k"]
        train = kind == "linear_train"
        s["x"] = randn(m, k).requires_grad_(train)
        s["w"] = randn(n, k, std=k**-0.5).requires_grad_(train)
        s["b"] = randn(n, std=0.5).requires_grad_(train) if case["bias"] else None
        s["r"] = randn(m, n).requires_grad_(train) if case["residual"] else None
        if train:
            s["dout"] = randn(m, n)
    else:
        B, H, D = case["batch"], case["heads"], case["head_dim"]
        train = kind == "attn_train"
        s["q"] = randn(B, case["q_len"], H, D, std=D**-0.5 if case["unit_scale"] else 1.0).requires_grad_(train)
        s["k"] = randn(B, case["k_len"], H, D).requires_grad_(train)
        s["v"] = randn(B, case["k_len"], H, D).requires_grad_(train)
        s["table"] = randn(case["buckets"], H).requires_grad_(train)
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
        if train:
            s["dout"] = randn(B, case["q_len"], H, D)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    ops = _ops()
    c = s["case"]
    kind = c["kind"]
    if kind in ("bias", "bias_grad"):
        pos = dict(bidirectional=c["bidirectional"], max_distance=c["max_distance"], q_offset=c["q_offset"])
        if kind == "bias":
            return ops.rel_pos_bias(s["table"], c["q_len"], c["k_len"], **pos)
        return ops.rel_pos_bias_grad(s["dbias"], c["buckets"], **pos)
    if kind in ("linear", "linear_train"):
        out = ops.linear_act_residual(s["x"], s["w"], s["b"], act=c["act"], residual=s["r"])
        if kind == "linear":
            return out
        leaves = [t for t in (s["x"], s["w"], s["b"], s["r"]) if t is not None]
        return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]
    out = ops.rel_pos_attention(s["q"], s["k"], s["v"], s["table"], k_lens=s["lens"], scale=_scale(c),
                                causal=c["causal"], bidirectional=c["bidirectional"],
                                max_distance=c["max_distance"], q_offset=c["q_offset"])
    if kind == "attn":
        return out
    return [out.detach(), *torch.autograd.grad(out, [s["q"], s["k"], s["v"], s["table"]], s["dout"])]


def _act(x, act):
    if act == "relu":
        return x.clamp_min(0)
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "gelu":
        return 0.5 * x * torch.erfc(-x * math.sqrt(0.5))
    if act == "gelu_tanh":
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x**3))
    return x


def _dact(x, act):
    if act == "relu":
        return (x > 0).to(x.dtype)
    if act == "silu":
        sg = torch.sigmoid(x)
        return sg * (1 + x * (1 - sg))
    if act == "gelu":
        return 0.5 * torch.erfc(-x * math.sqrt(0.5)) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a = 2 * math.sqrt(2 / math.pi)
        sg = torch.sigmoid(a * (x + 0.044715 * x**3))
        return sg + x * sg * (1 - sg) * a * (1 + 3 * 0.044715 * x * x)
    return torch.ones_like(x)


@torch.no_grad()
def _run_plain(s):
    c = s["case"]
    kind = c["kind"]
    dt = _DT[c["dtype"]]
    if kind == "bias":
        return s["table"].float()[_buckets(c, "cuda")].permute(2, 0, 1).to(dt).contiguous()
    if kind == "bias_grad":
        per_pos = s["dbias"].float().sum(0).flatten(1)  # [H, Lq * Lk]
        idx = _buckets(c, "cuda").flatten()
        out = torch.zeros(c["buckets"], c["heads"], device="cuda")
        for b in range(c["buckets"]):
            out[b] = per_pos[:, idx == b].sum(1)
        return out
    if kind in ("linear", "linear_train"):
        x, w = s["x"].float(), s["w"].float()
        pre = x @ w.T
        if s["b"] is not None:
            pre = pre + s["b"].float()
        out = _act(pre, c["act"])
        if s["r"] is not None:
            out = out + s["r"].float()
        if kind == "linear":
            return out.to(dt)
        dpre = s["dout"].float() * _dact(pre, c["act"])
        grads = [dpre @ w, dpre.T @ x]
        if s["b"] is not None:
            grads.append(dpre.sum(0))
        if s["r"] is not None:
            grads.append(s["dout"].float())
        return [out.to(dt), *[t.to(dt) for t in grads]]
    q, k, v = (s[n].float().transpose(1, 2) for n in ("q", "k", "v"))  # [B, H, L, D]
    bucket = _buckets(c, "cuda")
    j = torch.arange(c["k_len"], device="cuda")
    seen = (j[None, :] < s["lens"][:, None])[:, None, None, :]
    if c["causal"]:
        i = torch.arange(c["q_len"], device="cuda") + c["q_offset"]
        seen = seen & (j[None, :] <= i[:, None])
    score = (q @ k.transpose(-1, -2)).mul_(_scale(c)).add_(s["table"].float().T[:, bucket])
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    o = p @ v
    out = o.transpose(1, 2).to(dt).contiguous()
    if kind == "attn":
        return out
    do = s["dout"].float().transpose(1, 2)
    dv = p.transpose(-1, -2) @ do
    ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
    dq = ds @ k * _scale(c)
    dk = ds.transpose(-1, -2) @ q * _scale(c)
    per_pos = ds.sum(0).flatten(1)
    dtable = torch.zeros(c["buckets"], c["heads"], device="cuda")
    for b in range(c["buckets"]):
        dtable[b] = per_pos[:, (bucket == b).flatten()].sum(1)
    return [out, *[t.transpose(1, 2).to(dt).contiguous() for t in (dq, dk, dv)], dtable.to(dt)]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _pairs(case):
    """Visible (query, key) pairs of one head, all samples."""
    total = 0
    for n in _lens(case):
        if not case["causal"]:
            total += case["q_len"] * n
        else:
            first = min(n, case["q_offset"] + 1)  # keys the first query sees
            rise = min(case["q_len"], n - first)  # queries that each see one more
            total += case["q_len"] * first + rise * (rise - 1) // 2 + (case["q_len"] - rise) * rise
    return total


def work(case):
    e = _SIZE[case["dtype"]]
    kind = case["kind"]
    if kind in ("bias", "bias_grad"):
        cells = case["heads"] * case["q_len"] * case["k_len"] * case.get("batch", 1)
        small = case["buckets"] * case["heads"] * (e if kind == "bias" else 4)
        return {"bytes": cells * e + small, "flops": cells if kind == "bias_grad" else 0}
    if kind in ("linear", "linear_train"):
        m, n, k = case["m"], case["n"], case["k"]
        mats = m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)
        if kind == "linear":
            return {"bytes": mats * e, "flops": 2 * m * n * k}
        back = m * n + m * k + n * k + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        return {"bytes": (mats + back) * e, "flops": 6 * m * n * k}
    H, D = case["heads"], case["head_dim"]
    q = case["batch"] * case["q_len"] * H * D
    kv = 2 * sum(_lens(case)) * H * D
    table = case["buckets"] * H
    pairs = _pairs(case) * H
    if kind == "attn":
        return {"bytes": (2 * q + kv + table) * e, "flops": 4 * pairs * D}
    dkv = 2 * case["batch"] * case["k_len"] * H * D
    return {"bytes": (4 * q + kv + dkv + 2 * table) * e, "flops": 14 * pairs * D}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
@lru_cache(maxsize=None)
def _bucket_of(d, buckets, max_distance, bidirectional):
    """The bucket of relative position d = key - query, from the rule itself."""
    base, nb, n = 0, buckets, max(-d, 0)
    if bidirectional:
        nb = buckets // 2
        base, n = (nb if d > 0 else 0), abs(d)
    exact = nb // 2
    if n < exact:
        return base + n
    T = nb - exact
    t = 0  # the largest t < T with (n / exact)^T >= (max_distance / exact)^t
    while t + 1 < T and n**T * exact ** (t + 1) >= max_distance ** (t + 1) * exact**T:
        t += 1
    return base + exact + t


def _bucket_row(case, lo, hi):
    """Buckets of the relative positions lo .. hi - 1."""
    clip = case["max_distance"] + 1  # constant from there on
    return torch.tensor([_bucket_of(max(-clip, min(clip, d)), case["buckets"], case["max_distance"],
                                    case["bidirectional"]) for d in range(lo, hi)], device="cuda")


def _bucket_map(case):
    """[q_len, k_len] buckets from one row of relative positions."""
    lq, lk, off = case["q_len"], case["k_len"], case["q_offset"]
    row = _bucket_row(case, -(lq - 1) - off, lk - off)
    i = torch.arange(lq, device="cuda")[:, None]
    return row[torch.arange(lk, device="cuda")[None, :] - i + lq - 1]


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    f64 = torch.float64
    if kind == "bias":
        return torch.stack([s["table"].to(f64)[:, h][_bucket_map(case)] for h in range(case["heads"])])
    if kind == "bias_grad":
        where = _bucket_map(case).flatten()
        out = torch.zeros(case["buckets"], case["heads"], dtype=f64, device="cuda")
        for h in range(case["heads"]):
            out[:, h].index_add_(0, where, s["dbias"][:, h].to(f64).sum(0).flatten())
        return out
    if kind in ("linear", "linear_train"):
        x, w = s["x"].to(f64), s["w"].to(f64)
        pre = torch.einsum("mk,nk->mn", x, w)
        if s["b"] is not None:
            pre += s["b"].to(f64)
        half = math.sqrt(0.5)
        c0, c1 = math.sqrt(2 / math.pi), 0.044715
        f, df = {
            "none": (lambda t: t, torch.ones_like),
            "relu": (lambda t: torch.where(t > 0, t, 0.0), lambda t: torch.where(t > 0, 1.0, 0.0).to(f64)),
            "silu": (lambda t: t / (1 + torch.exp(-t)),
                     lambda t: (1 + torch.exp(-t) + t * torch.exp(-t)) / (1 + torch.exp(-t)) ** 2),
            "gelu": (lambda t: 0.5 * t * (1 + torch.erf(t * half)),
                     lambda t: 0.5 * (1 + torch.erf(t * half)) + t * torch.exp(-t * t / 2) / math.sqrt(2 * math.pi)),
            "gelu_tanh": (lambda t: 0.5 * t * (1 + torch.tanh(c0 * (t + c1 * t**3))),
                          lambda t: 0.5 * (1 + torch.tanh(c0 * (t + c1 * t**3)))
                          + 0.5 * t * (1 - torch.tanh(c0 * (t + c1 * t**3)) ** 2) * c0 * (1 + 3 * c1 * t * t)),
        }[case["act"]]
        out = f(pre)
        if s["r"] is not None:
            out += s["r"].to(f64)
        if kind == "linear":
            return out
        dpre = s["dout"].to(f64) * df(pre)
        grads = [torch.einsum("mn,nk->mk", dpre, w), torch.einsum("mn,mk->nk", dpre, x)]
        if s["b"] is not None:
            grads.append(dpre.sum(0))
        if s["r"] is not None:
            grads.append(s["dout"].to(f64))
        return [out, *grads]
    where = _bucket_map(case)
    lens = _lens(case)
    lq, lk, scale = case["q_len"], case["k_len"], _scale(case)
    train = kind == "attn_train"
    q, k, v = s["q"], s["k"], s["v"]
    res = [torch.zeros(t.shape, dtype=f64, device="cuda") for t in ((q, q, k, v, s["table"]) if train else (q,))]
    rows = torch.arange(lq, device="cuda")[:, None] + case["q_offset"]
    cols = torch.arange(lk, device="cuda")[None, :]
    for b, n in enumerate(lens):
        if n == 0:
            continue
        for h in range(case["heads"]):
            qh, kh, vh = q[b, :, h].to(f64), k[b, :n, h].to(f64), v[b, :n, h].to(f64)
            z = scale * torch.einsum("id,jd->ij", qh, kh) + s["table"][:, h].to(f64)[where[:, :n]]
            if case["causal"]:
                z = torch.where(cols[:, :n] <= rows, z, -math.inf)
            p = torch.softmax(z, -1)
            o = torch.einsum("ij,jd->id", p, vh)
            res[0][b, :, h] = o
            if not train:
                continue
            g = s["dout"][b, :, h].to(f64)
            dp = torch.einsum("id,jd->ij", g, vh)
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            res[1][b, :, h] = scale * torch.einsum("ij,jd->id", ds, kh)
            res[2][b, :n, h] = scale * torch.einsum("ij,id->jd", ds, qh)
            res[3][b, :n, h] = torch.einsum("ij,id->jd", p, g)
            res[4][:, h].index_add_(0, where[:, :n].flatten(), ds.flatten())
    return res if train else res[0]
