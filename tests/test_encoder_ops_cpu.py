"""Host logic of the text-encoder operators: bucket bounds, refusals (no device needed)."""
import ctypes

import pytest
import torch


def bucket(d, num_buckets, max_distance, bidirectional):
    base, nb, n = 0, num_buckets, max(-d, 0)
    if bidirectional:
        nb = num_buckets // 2
        base, n = (nb if d > 0 else 0), abs(d)
    exact = nb // 2
    if n < exact:
        return base + n
    T, t = nb - exact, 0
    while t + 1 < T and n**T * exact ** (t + 1) >= max_distance ** (t + 1) * exact**T:
        t += 1
    return base + exact + t


@pytest.mark.parametrize("nb,md,bi", [(32, 128, True), (32, 128, False), (16, 100, True), (2, 3, False),
                                      (8, 5, True), (4, 1000, True), (64, 500, True), (33, 200, False)])
def test_bounds_count_to_the_bucket(pkg, nb, md, bi):
    bounds = pkg.ops.rel_pos_bounds(nb, md, bi)
    one = nb // 2 if bi else nb
    assert len(bounds) == one - 1 and list(bounds) == sorted(bounds)
    for d in range(-2 * md, 2 * md):
        n = abs(d) if bi else max(-d, 0)
        b = sum(x <= n for x in bounds) + (one if bi and d > 0 else 0)
        assert b == bucket(d, nb, md, bi), d


def test_bounds_of_powers_fall_on_the_border(pkg):
    # 16 and 64 are exactly 2 and 6 of the 8 logarithmic steps from 8 to 128
    assert pkg.ops.rel_pos_bounds(32, 128, True) == (1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91)


def test_positions_refused(pkg):
    ops = pkg.ops
    with pytest.raises(ValueError, match="even number"):
        ops.rel_pos_bounds(31, 128, True)
    with pytest.raises(ValueError, match="max_distance"):
        ops.rel_pos_bounds(32, 8, True)
    with pytest.raises(ValueError, match="buckets a direction"):
        ops.rel_pos_bounds(1, 8, False)
    with pytest.raises(ValueError, match="buckets a direction"):
        ops.rel_pos_bounds(1024, 8000, True)
    t = torch.zeros(32, 4)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.rel_pos_bias(t, 4, 4)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.rel_pos_bias_grad(torch.zeros(4, 5, 6), 32)
    with pytest.raises(ValueError, match="negative"):
        ops.rel_pos_bias(t, 4, 4, q_offset=-1)
    with pytest.raises(ValueError, match="num_buckets, heads"):
        ops.rel_pos_bias(torch.zeros(32), 4, 4)
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        ops.rel_pos_bias(torch.zeros(32, 4, dtype=torch.float64), 4, 4)


def test_rel_pos_entry_points_validate_without_device(pkg):
    lib = pkg._lib.load()
    null, d = ctypes.c_void_p(None), ctypes.c_void_p(0x1000)
    bounds = (ctypes.c_int * 3)(1, 2, 8)
    down = (ctypes.c_int * 3)(1, 8, 2)

    def bias(table=d, dtype=0, b=bounds, n=3, H=2, Lq=4, Lk=4, off=0, out=d):
        return lib.wdit_rel_pos_bias(table, dtype, b, n, 1, H, Lq, Lk, off, out, null)

    assert bias(table=null) == 1 and bias(out=null) == 1 and bias(b=None) == 1 and bias(dtype=3) == 1
    assert bias(b=down) == 1
    assert bias(n=0) == 2 and bias(n=256) == 2 and bias(H=0) == 2 and bias(off=-1) == 2
    assert bias(Lq=-1) == 2 and bias(off=(1 << 30)) == 2
    assert bias(out=ctypes.c_void_p(0x1008)) == 3
    assert bias(table=null, out=null, Lq=0) == 0 and bias(table=null, out=null, Lk=0) == 0

    def grad(db=d, dtype=0, B=1, H=2, Lq=4, Lk=4, sb=32, b=bounds, n=3, off=0, out=d, ws=d, nbytes=1 << 20):
        return lib.wdit_rel_pos_bias_grad(db, dtype, B, H, Lq, Lk, sb, 16, 4, b, n, 1, off, out, ws, nbytes, null)

    assert grad(db=null) == 1 and grad(out=null) == 1 and grad(b=None) == 1 and grad(dtype=-1) == 1
    assert grad(b=down) == 1
    assert grad(n=0) == 2 and grad(B=-1) == 2 and grad(sb=-32) == 2
    assert grad(ws=null) == 5 and grad(nbytes=4) == 5
    assert grad(ws=ctypes.c_void_p(0x1004)) == 3
    assert lib.wdit_rel_pos_bias_grad_workspace_bytes(0, 2, 4, 4, 3, 1) == 0
    assert lib.wdit_rel_pos_bias_grad_workspace_bytes(1, 2, 4, 4, 3, 1) == 4 * 1 * 2 * 8
