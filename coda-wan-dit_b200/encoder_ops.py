"""Operators of the text encoder whose output the DiT's cross-attention reads.

* ``rel_pos_bias`` / ``rel_pos_bias_grad``: a learned relative position bias by buckets and the
  gradient of its table.

Public names are re-exported by ``ops``, beside the GEMM and position-table ops of the block.
Differentiable ops take part in autograd (first order); the others do not.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, ptr, stream_ptr

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_BUCKETS = 256  # table rows of one direction (kMaxRelBounds + 1 in csrc/relpos.cuh)


def _require_cuda(*ts: torch.Tensor | None) -> torch.device:
    """The tensors' common device."""
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("wdit ops run on CUDA tensors only (no CPU implementation)")
        if dev is not None and t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} and {t.device}")
        dev = t.device
    return dev


def _workspace(nbytes: int, device) -> torch.Tensor | None:
    # From torch's caching allocator on the current stream: calls never share one, and a captured
    # graph keeps its own.
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


# ---------------------------------------------------------------------------
# Relative position buckets
# ---------------------------------------------------------------------------
@lru_cache(maxsize=64)
def rel_pos_bounds(num_buckets: int, max_distance: int, bidirectional: bool) -> tuple[int, ...]:
    """Distances at which the bucket steps up by one (the bucket of distance n is the number of
    bounds <= n): one per distance below `exact` = half of a direction's buckets, then
    logarithmic up to max_distance. Bucket exact + t begins at the least n with
    log(n / exact) / log(max_distance / exact) * T >= t, T = buckets - exact, decided in whole
    numbers as n^T >= max_distance^t * exact^(T - t)."""
    if bidirectional and num_buckets % 2 != 0:
        raise ValueError(f"a bidirectional table needs an even number of buckets, got {num_buckets}")
    nb = num_buckets // 2 if bidirectional else num_buckets
    if not 2 <= nb <= MAX_BUCKETS:
        raise ValueError(f"2 to {MAX_BUCKETS} buckets a direction, got {nb}")
    exact = nb // 2
    if not exact < max_distance <= 1 << 30:
        raise ValueError(f"max_distance must be above {exact} (the exact distances) and at most 2^30, got {max_distance}")
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
    if q_len + q_offset > 1 << 30 or k_len > 1 << 30:
        raise ValueError("positions above 2^30")


def _check_table(table: torch.Tensor) -> None:
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError(f"table must be [num_buckets, heads], got {tuple(table.shape)}")
    if table.dtype not in _DTYPE:
        raise ValueError(f"table must be fp32, bf16 or fp16, got {table.dtype}")


def _rel_pos_bias(table, q_len, k_len, bidirectional, max_distance, q_offset):
    H = table.shape[1]
    bounds, n = _bounds_arg(table.shape[0], max_distance, bidirectional)
    with torch.cuda.device(table.device):
        table = table.contiguous()
        out = torch.empty((H, q_len, k_len), dtype=table.dtype, device=table.device)
        call("wdit_rel_pos_bias", ptr(table), _DTYPE[table.dtype], bounds, n, int(bidirectional), H, q_len, k_len,
             q_offset, ptr(out), stream_ptr())
    return out


def rel_pos_bias_grad(dbias: torch.Tensor, num_buckets: int, *, bidirectional: bool = True, max_distance: int = 128,
                      q_offset: int = 0) -> torch.Tensor:
    """Gradient of rel_pos_bias's table: dtable [num_buckets, H] fp32, the sum of the cells of
    dbias ([H, Lq, Lk], or [B, H, Lq, Lk] summed over the batch the bias was broadcast to; fp32,
    bf16 or fp16) by their bucket. Sums are fp32 in a fixed order: results repeat bit for bit."""
    dev = _require_cuda(dbias)
    if dbias.dim() == 3:
        dbias = dbias.unsqueeze(0)
    if dbias.dim() != 4:
        raise ValueError(f"dbias must be [H, Lq, Lk] or [B, H, Lq, Lk], got {tuple(dbias.shape)}")
    if dbias.dtype not in _DTYPE:
        raise ValueError(f"dbias must be fp32, bf16 or fp16, got {dbias.dtype}")
    B, H, Lq, Lk = dbias.shape
    if H < 1:
        raise ValueError("dbias has no heads")
    _check_positions(Lq, Lk, q_offset)
    bounds, n = _bounds_arg(num_buckets, max_distance, bidirectional)
    if dbias.stride(3) != 1 and Lk > 1:
        dbias = dbias.contiguous()
    with torch.cuda.device(dev):
        out = torch.empty((num_buckets, H), dtype=torch.float32, device=dev)
        nbytes = call("wdit_rel_pos_bias_grad_workspace_bytes", B, H, Lq, Lk, n, int(bidirectional))
        ws = _workspace(nbytes, dev)
        call("wdit_rel_pos_bias_grad", ptr(dbias), _DTYPE[dbias.dtype], B, H, Lq, Lk, dbias.stride(0), dbias.stride(1),
             dbias.stride(2), bounds, n, int(bidirectional), q_offset, ptr(out), ptr(ws), nbytes, stream_ptr(),
             kernels=2)
    return out


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
                                   q_offset=q_offset)
        return dtable.to(dtype), None, None, None, None, None


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
    if torch.is_grad_enabled() and table.requires_grad:
        return _RelPosBias.apply(table, q_len, k_len, bidirectional, max_distance, q_offset)
    return _rel_pos_bias(table, q_len, k_len, bidirectional, max_distance, q_offset)
