"""Operators of the text encoder whose output the DiT's cross-attention reads.

* ``rel_pos_bias`` / ``rel_pos_bias_grad``: a learned relative position bias by buckets and the
  gradient of its table.
* ``rel_pos_attention``: attention that reads that bias from its table, with its gradients.
* ``linear_act_residual``: act(x W^T + bias) + residual in one kernel, with its gradients.

Public names are re-exported by ``ops``, beside the GEMM and position-table ops of the block.
Differentiable ops take part in autograd (first order, reverse mode); forward-mode derivatives are
refused.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from operator import index

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import call, ptr

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_BUCKETS = 256  # table rows of one direction (kMaxRelBounds + 1 in csrc/relpos.cuh)
MAX_HEADS = 65535
MAX_LENGTH = 1 << 28  # queries or keys
MAX_EXTENT = 1 << 30  # M, N and K of a product (kMaxExtent in csrc/linear.cu), samples


def _require_cuda(*ts: torch.Tensor | None) -> int:
    """Index of the tensors' common device."""
    dev = -1
    for t in ts:
        if t is None:
            continue
        i = t.get_device()
        if i < 0:  # (a device without an index: the CPU, meta)
            raise RuntimeError("wdit ops run on CUDA tensors only (no CPU implementation)")
        if i != dev:
            if not t.is_cuda:
                raise RuntimeError("wdit ops run on CUDA tensors only (no CPU implementation)")
            if dev >= 0:
                raise ValueError(f"tensors on different devices: cuda:{dev} and cuda:{i}")
            dev = i
    if dev < 0:
        raise RuntimeError("wdit ops run on CUDA tensors only (no CPU implementation)")
    return dev


def _refuse_tangents(*ts: torch.Tensor | None) -> None:
    """The ops have no forward-mode derivatives: a dual tensor's tangent would be lost silently."""
    if forward_ad._current_level >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("forward-mode derivatives are not implemented for the encoder ops")


class _on_device:
    """Makes a device current around a launch; free when it is already (torch.cuda.device is not:
    several microseconds a call)."""

    __slots__ = ("dev", "prev")

    def __init__(self, dev: int):
        self.dev = dev

    def __enter__(self):
        self.prev = torch.cuda.current_device()
        if self.prev != self.dev:
            torch.cuda.set_device(self.dev)

    def __exit__(self, *exc):
        if self.prev != self.dev:
            torch.cuda.set_device(self.prev)
        return False


def _stream(dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev)  # the handle without a Stream object


def _workspace(nbytes: int, device) -> torch.Tensor | None:
    # From torch's caching allocator on the current stream: calls never share one, and a captured
    # graph keeps its own.
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


@lru_cache(maxsize=512)
def _workspace_bytes(dev: int, name: str, *shape: int) -> int:
    """Workspace query of an entry point (a function of the shape and the device)."""
    return call(name, *shape)


# ---------------------------------------------------------------------------
# Relative position buckets
# ---------------------------------------------------------------------------
def rel_pos_bounds(num_buckets: int, max_distance: int, bidirectional: bool) -> tuple[int, ...]:
    """Distances at which the bucket steps up by one (the bucket of distance n is the number of
    bounds <= n): one per distance below `exact` = half of a direction's buckets, then
    logarithmic up to max_distance. Bucket exact + t begins at the least n with
    log(n / exact) / log(max_distance / exact) * T >= t, T = buckets - exact, decided in whole
    numbers as n^T >= max_distance^t * exact^(T - t)."""
    # (whole numbers before the cache, for which 128.0 is 128)
    return _rel_pos_bounds(index(num_buckets), index(max_distance), bool(bidirectional))


@lru_cache(maxsize=64)
def _rel_pos_bounds(num_buckets: int, max_distance: int, bidirectional: bool) -> tuple[int, ...]:
    if bidirectional and num_buckets % 2 != 0:
        raise ValueError(f"a bidirectional table needs an even number of buckets, got {num_buckets}")
    nb = num_buckets // 2 if bidirectional else num_buckets
    if not 2 <= nb <= MAX_BUCKETS:
        raise ValueError(f"2 to {MAX_BUCKETS} buckets a direction, got {nb}")
    exact = nb // 2
    if not exact < max_distance <= 1 << 29:
        raise ValueError(f"max_distance must be above {exact} (the exact distances) and at most 2^29, got {max_distance}")
    T = nb - exact
    bounds = list(range(1, exact + 1))
    for t in range(1, T):
        target = max_distance**t * exact ** (T - t)
        lo, hi = exact, max_distance
        while lo < hi:
            mid = (lo + hi) // 2
            if mid**T >= target:
                hi = mid
            else:
                lo = mid + 1
        bounds.append(lo)
    return tuple(bounds)


@lru_cache(maxsize=64)
def _bounds_arg(num_buckets: int, max_distance: int, bidirectional: bool):
    bounds = rel_pos_bounds(num_buckets, max_distance, bidirectional)
    return (ctypes.c_int * len(bounds))(*bounds), len(bounds)


def _check_positions(q_len: int, k_len: int, q_offset: int) -> None:
    if q_len < 0 or k_len < 0 or q_offset < 0:
        raise ValueError(f"negative length or offset: q_len {q_len}, k_len {k_len}, q_offset {q_offset}")
    if q_len > MAX_LENGTH or k_len > MAX_LENGTH or q_len + q_offset > 1 << 30:
        raise ValueError(f"lengths up to 2^28 and positions up to 2^30, got q_len {q_len}, k_len {k_len}, "
                         f"q_offset {q_offset}")


def _check_table(table: torch.Tensor) -> None:
    if table.dim() != 2 or not 1 <= table.shape[1] <= MAX_HEADS:
        raise ValueError(f"table must be [num_buckets, heads], 1 to {MAX_HEADS} heads, got {tuple(table.shape)}")
    if table.dtype not in _DTYPE:
        raise ValueError(f"table must be fp32, bf16 or fp16, got {table.dtype}")


def _rel_pos_bias(table, q_len, k_len, bidirectional, max_distance, q_offset):
    dev = table.get_device()
    nb, H = table.shape
    bounds, n = _bounds_arg(nb, max_distance, bidirectional)
    with _on_device(dev):
        table = table.contiguous()
        out = table.new_empty((H, q_len, k_len))
        call("wdit_rel_pos_bias", table.data_ptr(), _DTYPE[table.dtype], bounds, n, bidirectional, H, q_len, k_len,
             q_offset, out.data_ptr(), _stream(dev))
    return out


def _rel_pos_bias_grad(dbias, num_buckets, bidirectional, max_distance, q_offset, dtype):
    dev = dbias.get_device()
    B, H, Lq, Lk = dbias.shape
    bounds, n = _bounds_arg(num_buckets, max_distance, bidirectional)
    with _on_device(dev):
        if Lk > 1 and dbias.stride(3) != 1:
            dbias = dbias.contiguous()
        out = torch.empty((num_buckets, H), dtype=dtype, device=dbias.device)
        nbytes = _workspace_bytes(dev, "wdit_rel_pos_bias_grad_workspace_bytes", B, H, Lq, Lk, n, int(bidirectional))
        ws = _workspace(nbytes, dbias.device)
        sb, sh, si, _ = dbias.stride()
        call("wdit_rel_pos_bias_grad", dbias.data_ptr(), _DTYPE[dbias.dtype], B, H, Lq, Lk, sb, sh, si, bounds, n,
             bidirectional, q_offset, out.data_ptr(), _DTYPE[dtype], ptr(ws), nbytes, _stream(dev), kernels=2)
    return out


class _RelPosBiasGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dbias, num_buckets, bidirectional, max_distance, q_offset, dtype):
        ctx.args = (*dbias.shape[2:], bidirectional, max_distance, q_offset)
        ctx.batch, ctx.dtype = dbias.shape[0], dbias.dtype
        return _rel_pos_bias_grad(dbias, num_buckets, bidirectional, max_distance, q_offset, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        # a cell's gradient is its bucket's (rounded before it is copied to the cells)
        d = _rel_pos_bias(g.to(ctx.dtype), *ctx.args)
        return d.expand(ctx.batch, *d.shape), None, None, None, None, None


def rel_pos_bias_grad(dbias: torch.Tensor, num_buckets: int, *, bidirectional: bool = True, max_distance: int = 128,
                      q_offset: int = 0, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Gradient of rel_pos_bias's table: dtable [num_buckets, H], the sum of the cells of dbias
    ([H, Lq, Lk], or [B, H, Lq, Lk] summed over the batch the bias was broadcast to; fp32, bf16
    or fp16) by their bucket. Sums are fp32 in a fixed order (results repeat bit for bit) and
    rounded once to dtype (fp32, bf16 or fp16). Differentiable in dbias."""
    dev = _require_cuda(dbias)
    _refuse_tangents(dbias)
    if dbias.dim() == 3:
        dbias = dbias.unsqueeze(0)
    if dbias.dim() != 4:
        raise ValueError(f"dbias must be [H, Lq, Lk] or [B, H, Lq, Lk], got {tuple(dbias.shape)}")
    if dbias.dtype not in _DTYPE:
        raise ValueError(f"dbias must be fp32, bf16 or fp16, got {dbias.dtype}")
    if dtype not in _DTYPE:
        raise ValueError(f"dtype must be fp32, bf16 or fp16, got {dtype}")
    B, H, Lq, Lk = dbias.shape
    if not 1 <= H <= MAX_HEADS or B > MAX_EXTENT:
        raise ValueError(f"1 to {MAX_HEADS} heads and at most 2^30 samples, got {H} and {B}")
    _check_positions(Lq, Lk, q_offset)
    if torch.is_grad_enabled() and dbias.requires_grad:
        return _RelPosBiasGrad.apply(dbias, num_buckets, bidirectional, max_distance, q_offset, dtype)
    return _rel_pos_bias_grad(dbias, num_buckets, bidirectional, max_distance, q_offset, dtype)


class _RelPosBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, q_len, k_len, bidirectional, max_distance, q_offset):
        ctx.args = (table.shape[0], table.dtype, bidirectional, max_distance, q_offset)
        return _rel_pos_bias(table, q_len, k_len, bidirectional, max_distance, q_offset)

    @staticmethod
    @once_differentiable
    def backward(ctx, dbias):
        num_buckets, dtype, bidirectional, max_distance, q_offset = ctx.args
        dtable = rel_pos_bias_grad(dbias, num_buckets, bidirectional=bidirectional, max_distance=max_distance,
                                   q_offset=q_offset, dtype=dtype)
        return dtable, None, None, None, None, None


def rel_pos_bias(table: torch.Tensor, q_len: int, k_len: int, *, bidirectional: bool = True, max_distance: int = 128,
                 q_offset: int = 0) -> torch.Tensor:
    """bias [H, q_len, k_len] of table's dtype: bias[h, i, j] = table[bucket(j - (i + q_offset)), h].

    table [num_buckets, H] (fp32, bf16 or fp16). bidirectional: keys ahead of the query take the
    upper half of the buckets; otherwise they share bucket 0 with the query itself. q_offset is
    the position of the first query (one token after a cache of n keys: q_len 1, q_offset n).
    Differentiable in table (rel_pos_bias_grad)."""
    _check_table(table)
    _check_positions(q_len, k_len, q_offset)
    rel_pos_bounds(table.shape[0], max_distance, bidirectional)  # refuses what the rule does not cover
    _require_cuda(table)
    _refuse_tangents(table)
    if torch.is_grad_enabled() and table.requires_grad:
        return _RelPosBias.apply(table, q_len, k_len, bidirectional, max_distance, q_offset)
    return _rel_pos_bias(table, q_len, k_len, bidirectional, max_distance, q_offset)


# ---------------------------------------------------------------------------
# act(x W^T + bias) + residual
# ---------------------------------------------------------------------------
_ACT = {"none": 0, "gelu_tanh": 1, "relu": 2, "silu": 3, "gelu": 4}


def _rows(t: torch.Tensor, cols: int) -> tuple[torch.Tensor, int, int]:
    """2-D operand of `cols` (a multiple of 8) columns with its pointer and row stride, as the
    kernels take it (unit column stride, rows on 16-byte boundaries), or a contiguous copy."""
    p = t.data_ptr()
    if p & 15 == 0:
        if t.is_contiguous():
            return t, p, cols
        ld, one = t.stride()
        if one == 1 and (t.shape[0] <= 1 or (ld % 8 == 0 and ld >= cols)):
            return t, p, ld if t.shape[0] > 1 else cols  # a single row's stride says nothing
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), cols


def _product(dev, dtype, a, a_mn, b, b_mn, M, N, K, out, bias=None, act=0, res=None, pre=None):
    """a, b, res as _rows gives them."""
    _, pa, lda = a
    _, pb, ldb = b
    pr, ldr = (None, 0) if res is None else res[1:]
    call("wdit_linear_act_residual", pa, lda, a_mn, pb, ldb, b_mn, M, N, K, _DTYPE[dtype],
         None if bias is None else bias.data_ptr(), 0 if bias is None else _DTYPE[bias.dtype], act, pr, ldr,
         out.data_ptr(), N, None if pre is None else pre.data_ptr(), N, _stream(dev))


def _linear_forward(dev, x, w, bias, act, residual, out, pre):
    N, K = w.shape
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if residual is not None:
        residual = _rows(residual if residual.dim() == 2 else residual.reshape(-1, N), N)
    if bias is not None and bias.stride(0) != 1:
        bias = bias.contiguous()
    _product(dev, x.dtype, _rows(x2, K), 0, _rows(w, K), 0, x2.shape[0], N, K, out, bias, _ACT[act], residual, pre)


class _LinearActResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, act, residual):
        dev = x.get_device()
        with _on_device(dev):
            out = x.new_empty((*x.shape[:-1], w.shape[0]))
            # The derivative needs pre = x W^T + bias: kept in the operands' type (half a step of
            # it moves act' by no more than rounding the gradient itself does).
            need = any(ctx.needs_input_grad[:3]) and act != "none"
            pre = torch.empty_like(out) if need else None
            _linear_forward(dev, x, w, bias, act, residual, out, pre)
        ctx.save_for_backward(x, w, pre)
        ctx.act = act
        ctx.bias_dtype = None if bias is None else bias.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, w, pre = ctx.saved_tensors
        need_x, need_w, need_b, _, need_r = ctx.needs_input_grad
        N, K = w.shape
        x2 = x if x.dim() == 2 else x.reshape(-1, K)
        M = x2.shape[0]
        dx = dw = db = None
        dev = x.get_device()
        with _on_device(dev):
            if need_x or need_w or need_b:
                g = _rows(dout if dout.dim() == 2 else dout.reshape(-1, N), N)
                dpre = g
                if pre is not None:
                    t = x.new_empty((M, N))
                    dpre = (t, t.data_ptr(), N)
                ws, nbytes = None, 0
                if need_b:
                    db = x.new_empty(N, dtype=ctx.bias_dtype)
                    nbytes = _workspace_bytes(dev, "wdit_act_backward_workspace_bytes", M, N)
                    ws = _workspace(nbytes, x.device)
                if need_b or pre is not None:
                    call("wdit_act_backward", g[1], g[2], ptr(pre), N, _ACT[ctx.act] if pre is not None else 0,
                         _DTYPE[x.dtype], M, N, dpre[1], dpre[2], ptr(db), 0 if db is None else _DTYPE[db.dtype],
                         ptr(ws), nbytes, _stream(dev), kernels=2 if nbytes > 0 else 1)
                if need_x:
                    dx = x.new_empty((M, K))
                    _product(dev, x.dtype, dpre, 0, _rows(w, K), 1, M, K, N, dx)
                    if x.dim() != 2:
                        dx = dx.view(x.shape)
                if need_w:
                    if M == 0:
                        dw = torch.zeros((N, K), dtype=w.dtype, device=w.device)
                    else:
                        dw = w.new_empty((N, K))
                        _product(dev, x.dtype, dpre, 1, _rows(x2, K), 1, N, K, M, dw)
        return dx, dw, db, None, dout if need_r else None


def linear_act_residual(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *, act: str = "none",
                        residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """act(x @ w.T + bias) + residual in one kernel, summed in fp32 and rounded once.

    x [..., K] and w [N, K] (nn.Linear.weight) bf16 or fp16, N and K multiples of 8; bias [N] of
    fp32, bf16 or fp16; residual [..., N] and out of x's dtype; act one of "none", "relu",
    "silu", "gelu" (erf), "gelu_tanh". Any number of rows, one included. out (contiguous; may be
    the residual itself) is for calls outside autograd. Differentiable in x, w, bias and
    residual. Operands whose rows do not start on 16-byte boundaries are copied first."""
    if act not in _ACT:
        raise ValueError(f"unknown activation {act!r} ({', '.join(_ACT)})")
    xs, ws = x.shape, w.shape
    if len(xs) < 1 or len(ws) != 2 or xs[-1] != ws[1]:
        raise ValueError(f"x [..., K] and w [N, K] expected, got {tuple(xs)} and {tuple(ws)}")
    dtype = x.dtype
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or w.dtype is not dtype:
        raise ValueError(f"x and w must both be bf16 or both fp16, got {x.dtype} and {w.dtype}")
    N, K = ws
    if N % 8 != 0 or K % 8 != 0 or N == 0 or K == 0:
        raise ValueError(f"N and K must be multiples of 8, got N {N}, K {K}")
    if N > MAX_EXTENT or K > MAX_EXTENT or x.numel() // K > MAX_EXTENT:
        raise ValueError(f"at most 2^30 rows, N and K, got {x.numel() // K}, {N} and {K}")
    shape = (*xs[:-1], N)
    if bias is not None and (bias.shape != (N,) or bias.dtype not in _DTYPE):
        raise ValueError(f"bias must be [{N}] of fp32, bf16 or fp16, got {tuple(bias.shape)} {bias.dtype}")
    if residual is not None and (residual.shape != shape or residual.dtype is not dtype):
        raise ValueError(f"residual must be {shape} of {dtype}, got {tuple(residual.shape)} {residual.dtype}")
    if out is not None and (out.shape != shape or out.dtype is not dtype):
        raise ValueError(f"out must be {shape} of {dtype}, got {tuple(out.shape)} {out.dtype}")
    dev = _require_cuda(x, w, bias, residual, out)
    _refuse_tangents(x, w, bias, residual)
    if torch.is_grad_enabled() and (
            x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad)
            or (residual is not None and residual.requires_grad) or (out is not None and out.requires_grad)):
        if out is not None:
            raise ValueError("out= is not supported where a gradient is recorded")
        return _LinearActResidual.apply(x, w, bias, act, residual)
    with _on_device(dev):
        if out is None:
            out = x.new_empty(shape)
        else:
            if not out.is_contiguous() or out.data_ptr() % 16 != 0:
                raise ValueError("out must be contiguous and start on a 16-byte boundary")
            _check_out_overlap(out, residual, x, w, bias)
            increment_version(out)  # autograd sees that it was written
        _linear_forward(dev, x, w, bias, act, residual, out, None)
    return out


def _extent(t: torch.Tensor) -> tuple[int, int]:
    if t.numel() == 0:
        return (t.data_ptr(), t.data_ptr())
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return (t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size())


def _check_out_overlap(out, residual, *inputs) -> None:
    """out may be exactly the residual (every element is read before it is written); any other
    overlap with an input would be read after it was overwritten."""
    lo, hi = _extent(out)
    for t in inputs:
        if t is not None:
            a, b = _extent(t)
            if a < hi and lo < b:
                raise ValueError("out overlaps an operand")
    if residual is not None:
        a, b = _extent(residual)
        same = residual.data_ptr() == out.data_ptr() and residual.stride() == out.stride()
        if a < hi and lo < b and not same:
            raise ValueError("out partly overlaps the residual")


# ---------------------------------------------------------------------------
# Attention with the relative position bias
# ---------------------------------------------------------------------------
def _heads(t: torch.Tensor) -> torch.Tensor:
    """[B, L, H, D] the kernels take as it is (unit stride along D, the other strides positive
    multiples of 8 elements, 16-byte aligned), or a contiguous copy."""
    if t.is_contiguous() and t.data_ptr() & 15 == 0:
        return t
    (B, L, H, _), (sb, sl, sh, sd) = t.shape, t.stride()
    if (sd == 1 and t.data_ptr() % 16 == 0 and (B == 1 or (sb > 0 and sb % 8 == 0))
            and (L == 1 or (sl > 0 and sl % 8 == 0)) and (H == 1 or (sh > 0 and sh % 8 == 0))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


@lru_cache(maxsize=1024)
def _strides_arg(B: int, L: int, H: int, D: int, sb: int, sl: int, sh: int, _: int):
    # a dimension of size 1 has no meaningful stride; any valid one does
    return (ctypes.c_longlong * 3)(sb if B > 1 else D, sl if L > 1 else D, sh if H > 1 else D)


def _strides(t: torch.Tensor):
    return _strides_arg(*t.shape, *t.stride())


def _attention_args(q, k, table, k_lens, bidirectional, causal, max_distance, q_offset, scale):
    B, Lq, H, D = q.shape
    bounds, n = _bounds_arg(table.shape[0], max_distance, bidirectional)
    shape = (B, H, Lq, k.shape[1], D)
    pos = (_DTYPE[q.dtype], None if k_lens is None else k_lens.data_ptr(), table.data_ptr(), _DTYPE[table.dtype],
           bounds, n, bidirectional, causal, q_offset, scale)
    return shape, pos


def _attention_forward(dev, q, k, v, table, k_lens, bidirectional, causal, max_distance, q_offset, scale, for_grad):
    B, Lq, H, D = q.shape
    device = q.device
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if B == 0 or Lq == 0 or k.shape[1] == 0:
        return out.zero_(), None
    lse = torch.empty((B, H, Lq), dtype=torch.float32, device=device) if for_grad else None
    shape, pos = _attention_args(q, k, table, k_lens, bidirectional, causal, max_distance, q_offset, scale)
    nbytes = _workspace_bytes(dev, "wdit_rel_attention_workspace_bytes", *shape)
    ws = _workspace(nbytes, device)
    call("wdit_rel_attention", q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v), *shape,
         *pos, out.data_ptr(), ptr(lse), ptr(ws), nbytes, _stream(dev), kernels=1 if nbytes == 0 else 2)
    return out, lse


class _RelPosAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, k_lens, bidirectional, causal, max_distance, q_offset, scale):
        dev = q.get_device()
        with _on_device(dev):
            qc, kc, vc, tc = _heads(q), _heads(k), _heads(v), table.contiguous()
            out, lse = _attention_forward(dev, qc, kc, vc, tc, k_lens, bidirectional, causal, max_distance, q_offset,
                                          scale, True)
        ctx.save_for_backward(qc, kc, vc, tc, k_lens, lse)
        ctx.args = (bidirectional, causal, max_distance, q_offset, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, table, k_lens, lse = ctx.saved_tensors
        nothing = (None,) * 6
        if lse is None:  # no queries or no keys
            return (torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(table), *nothing)
        dev = q.get_device()
        with _on_device(dev):
            g = _heads(dout)
            device = q.device
            dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
            dtable = torch.empty_like(table)  # (contiguous)
            shape, pos = _attention_args(q, k, table, k_lens, *ctx.args)
            nbytes = _workspace_bytes(dev, "wdit_rel_attention_backward_workspace_bytes", *shape[:3], pos[5],
                                      int(pos[6]))
            ws = _workspace(nbytes, device)
            call("wdit_rel_attention_backward", q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(),
                 _strides(v), g.data_ptr(), _strides(g), lse.data_ptr(), *shape, *pos, dq.data_ptr(),
                 dk.data_ptr(), dv.data_ptr(), dtable.data_ptr(), _DTYPE[table.dtype], ws.data_ptr(), nbytes,
                 _stream(dev), kernels=3)
        return (dq, dk, dv, dtable, *nothing)


def rel_pos_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, *,
                      k_lens: torch.Tensor | None = None, scale: float | None = None, causal: bool = False,
                      bidirectional: bool = True, max_distance: int = 128, q_offset: int = 0) -> torch.Tensor:
    """softmax(scale q k^T + bias) v with rel_pos_bias's bias read from its table: [B, Lq, H, D].

    q [B, Lq, H, D], k and v [B, Lk, H, D] (bf16 or fp16, D 64 or 128; any strides, rows of a head
    contiguous and on 16-byte boundaries, others are copied); table [num_buckets, H] (fp32, bf16
    or fp16). k_lens [B] int32: sample b's first k_lens[b] keys are valid (clamped to [0, Lk]; what
    lies behind them is not looked at). causal: query i sees the keys up to i + q_offset (those past
    the last query may hold anything; an infinity or NaN of a key that some query sees may reach
    the queries before it too, as 0 times it). A row that sees no key gives 0. Finite table values
    past +-11356 count as +-11356: a mask of the type's lowest value leaves a key no weight beside
    others, and a row of nothing but such keys is the softmax of their scores; -inf hides a key. scale defaults to D ** -0.5. One token after a cache of n keys:
    Lq 1, q_offset n - 1 if the cache holds the token's own key, n otherwise. Differentiable in
    q, k, v and table; results repeat bit for bit."""
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape:
        raise ValueError(f"q [B, Lq, H, D], k and v [B, Lk, H, D] expected, got {tuple(qs)}, {tuple(ks)}, "
                         f"{tuple(v.shape)}")
    B, Lq, H, D = qs
    if B > MAX_EXTENT:
        raise ValueError(f"at most 2^30 samples, got {B}")
    if ks[0] != B or ks[2] != H or ks[3] != D:
        raise ValueError(f"q {tuple(qs)} and k {tuple(ks)} differ in batch, heads or head size")
    if D != 64 and D != 128:
        raise ValueError(f"head size 64 or 128, got {D}")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError(f"q, k and v must all be bf16 or all fp16, got {q.dtype}, {k.dtype}, {v.dtype}")
    _check_table(table)
    if table.shape[1] != H:
        raise ValueError(f"table for {table.shape[1]} heads, q has {H}")
    _check_positions(Lq, ks[1], q_offset)
    rel_pos_bounds(table.shape[0], max_distance, bidirectional)
    if k_lens is not None:
        if k_lens.shape != (B,) or k_lens.dtype is not torch.int32:
            raise ValueError(f"k_lens must be [{B}] int32, got {tuple(k_lens.shape)} {k_lens.dtype}")
        k_lens = k_lens.contiguous()
    dev = _require_cuda(q, k, v, table, k_lens)
    _refuse_tangents(q, k, v, table)
    scale = D**-0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or table.requires_grad):
        return _RelPosAttention.apply(q, k, v, table, k_lens, bidirectional, causal, max_distance, q_offset, scale)
    with _on_device(dev):
        return _attention_forward(dev, _heads(q), _heads(k), _heads(v), table.contiguous(), k_lens, bidirectional,
                                  causal, max_distance, q_offset, scale, False)[0]
