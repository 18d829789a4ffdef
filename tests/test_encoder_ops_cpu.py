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


def test_extents_refused(pkg):
    """Sizes past the kernels' 32-bit coordinates: refused, not wrapped (expanded tensors hold nothing)."""
    ops, big = pkg.ops, (1 << 28) + 1
    t = torch.zeros(32, 4)
    for lq, lk, off in [(big, 1, 0), (1, big, 0), (1, 1, 1 << 30)]:
        with pytest.raises(ValueError, match="lengths up to"):
            ops.rel_pos_bias(t, lq, lk, q_offset=off)
    with pytest.raises(ValueError, match="heads"):
        ops.rel_pos_bias(torch.zeros(1).expand(32, 65536), 4, 4)
    with pytest.raises(ValueError, match="at most 2\\^29"):
        ops.rel_pos_bias(t, 4, 4, max_distance=(1 << 29) + 1)
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        ops.rel_pos_bias(t.double(), 4, 4)
    half = torch.zeros(1, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="at most 2\\^30 rows"):
        ops.linear_act_residual(half.expand((1 << 30) + 1, 64), half.expand(8, 64))
    with pytest.raises(ValueError, match="at most 2\\^30 rows"):
        ops.linear_act_residual(half.expand(1, (1 << 30) + 8), half.expand(8, (1 << 30) + 8))
    q, k = half.expand(1, 4, 4, 64), half.expand(1, big, 4, 64)
    with pytest.raises(ValueError, match="lengths up to"):
        ops.rel_pos_attention(q, k, k, t)
    lib, null, d = pkg._lib.load(), ctypes.c_void_p(None), ctypes.c_void_p(0x1000)
    b = (ctypes.c_int * 1)(1)
    st = (ctypes.c_longlong * 3)(64, 64, 64)
    assert lib.wdit_rel_pos_bias(d, 0, b, 1, 1, 65536, 4, 4, 0, d, null) == 2
    assert lib.wdit_rel_pos_bias(d, 0, b, 1, 1, 4, 4, big, 0, d, null) == 2
    assert lib.wdit_linear_act_residual(d, 64, 0, d, 64, 0, (1 << 30) + 1, 64, 64, 1, null, 0, 0, null, 0, d, 64, null,
                                        0, null) == 2
    for H, lq, lk in [(65536, 1, 1), (1, big, 1), (1, 1, big)]:
        assert lib.wdit_rel_attention(d, st, d, st, d, st, 1, H, lq, lk, 64, 1, null, d, 0, b, 1, 1, 0, 0, 1.0, d, null,
                                      null, 0, null) == 2


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

    def grad(db=d, dtype=0, B=1, H=2, Lq=4, Lk=4, sb=32, b=bounds, n=3, off=0, out=d, ddt=0, ws=d, nbytes=1 << 20):
        return lib.wdit_rel_pos_bias_grad(db, dtype, B, H, Lq, Lk, sb, 16, 4, b, n, 1, off, out, ddt, ws, nbytes, null)

    assert grad(db=null) == 1 and grad(out=null) == 1 and grad(b=None) == 1 and grad(dtype=-1) == 1
    assert grad(b=down) == 1 and grad(ddt=3) == 1
    assert grad(n=0) == 2 and grad(B=-1) == 2 and grad(sb=-32) == 2
    assert grad(ws=null) == 5 and grad(nbytes=4) == 5
    assert grad(ws=ctypes.c_void_p(0x1004)) == 3
    assert lib.wdit_rel_pos_bias_grad_workspace_bytes(0, 2, 4, 4, 3, 1) == 0
    assert lib.wdit_rel_pos_bias_grad_workspace_bytes(1, 2, 4, 4, 3, 1) == 4 * 1 * 2 * 8


def test_linear_refused(pkg):
    f = pkg.ops.linear_act_residual
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        f(bf(4, 64), bf(32, 64))
    with pytest.raises(ValueError, match="unknown activation"):
        f(bf(4, 64), bf(32, 64), act="tanh")
    with pytest.raises(ValueError, match="expected"):
        f(bf(4, 64), bf(32, 72))
    with pytest.raises(ValueError, match="both be bf16 or both fp16"):
        f(bf(4, 64), bf(32, 64).half())
    with pytest.raises(ValueError, match="both be bf16 or both fp16"):
        f(torch.zeros(4, 64), torch.zeros(32, 64))
    for n, k in [(33, 64), (32, 60), (0, 64), (32, 0)]:
        with pytest.raises(ValueError, match="multiples of 8"):
            f(bf(4, k), bf(n, k))
    with pytest.raises(ValueError, match="bias must be"):
        f(bf(4, 64), bf(32, 64), bf(64))
    with pytest.raises(ValueError, match="residual must be"):
        f(bf(4, 64), bf(32, 64), residual=bf(1, 32))
    with pytest.raises(ValueError, match="out must be"):
        f(bf(4, 64), bf(32, 64), out=torch.zeros(4, 32))


def test_attention_refused(pkg):
    f = pkg.ops.rel_pos_attention
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    q, t = bf(2, 5, 3, 64), torch.zeros(32, 3)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        f(q, q, q, t)
    with pytest.raises(ValueError, match="expected"):
        f(q, q, bf(2, 6, 3, 64), t)
    with pytest.raises(ValueError, match="differ in batch"):
        f(q, bf(2, 5, 1, 64), bf(2, 5, 1, 64), t)
    with pytest.raises(ValueError, match="head size"):
        f(bf(2, 5, 3, 80), bf(2, 5, 3, 80), bf(2, 5, 3, 80), t)
    with pytest.raises(ValueError, match="all be bf16"):
        f(q, q.half(), q, t)
    with pytest.raises(ValueError, match="table for 4 heads"):
        f(q, q, q, torch.zeros(32, 4))
    with pytest.raises(ValueError, match="even number"):
        f(q, q, q, torch.zeros(31, 3))
    with pytest.raises(ValueError, match="k_lens must be"):
        f(q, q, q, t, k_lens=torch.zeros(2))
    with pytest.raises(ValueError, match="k_lens must be"):
        f(q, q, q, t, k_lens=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="negative"):
        f(q, q, q, t, q_offset=-1)


def test_linear_entry_points_validate_without_device(pkg):
    lib = pkg._lib.load()
    null, d = ctypes.c_void_p(None), ctypes.c_void_p(0x1000)

    def lin(A=d, lda=64, a_mn=0, B=d, ldb=64, b_mn=0, M=4, N=32, K=64, dtype=1, bias=d, bd=0, act=0, res=d, ldr=32,
            out=d, ldo=32, pre=null, ldp=0):
        return lib.wdit_linear_act_residual(A, lda, a_mn, B, ldb, b_mn, M, N, K, dtype, bias, bd, act, res, ldr, out,
                                            ldo, pre, ldp, null)

    assert lin(A=null) == 1 and lin(B=null) == 1 and lin(out=null) == 1
    assert lin(dtype=0) == 1 and lin(act=5) == 1 and lin(bd=3) == 1 and lin(a_mn=1) == 1
    assert lin(N=36) == 2 and lin(K=0) == 2 and lin(M=-1) == 2
    assert lin(lda=56) == 2 and lin(ldb=56) == 2 and lin(ldo=24) == 2 and lin(ldr=24) == 2
    assert lin(pre=d, ldp=24) == 2
    assert lin(lda=68) == 3 and lin(A=ctypes.c_void_p(0x1008)) == 3 and lin(res=ctypes.c_void_p(0x1002)) == 3
    assert lin(A=null, out=null, M=0) == 0

    def back(dout=d, pre=d, act=3, dtype=1, M=400, N=32, dpre=d, db=d, dbt=0, ws=d, nb=1 << 20, ld=32):
        return lib.wdit_act_backward(dout, ld, pre, ld, act, dtype, M, N, dpre, ld, db, dbt, ws, nb, null)

    assert back(dout=null) == 1 and back(pre=null) == 1 and back(dpre=null) == 1 and back(act=9) == 1
    assert back(dtype=0) == 1 and back(dbt=3) == 1
    assert back(N=30) == 2 and back(M=-1) == 2 and back(ld=24) == 2
    assert back(ld=36) == 3 and back(ws=null) == 5 and back(nb=16) == 5
    assert back(act=0, db=null, dout=null) == 0  # dpre is dout, no bias: nothing to do
    assert lib.wdit_act_backward_workspace_bytes(65, 32) == 4 * 2 * 32
    assert lib.wdit_act_backward_workspace_bytes(64, 32) == 0


def test_attention_entry_points_validate_without_device(pkg):
    lib = pkg._lib.load()
    null, d = ctypes.c_void_p(None), ctypes.c_void_p(0x1000)
    bounds = (ctypes.c_int * 3)(1, 2, 8)
    st = (ctypes.c_longlong * 3)(5 * 3 * 64, 3 * 64, 64)
    bad = (ctypes.c_longlong * 3)(5 * 3 * 64, 3 * 64 + 4, 64)
    zero = (ctypes.c_longlong * 3)(5 * 3 * 64, 0, 64)

    def fwd(q=d, qs=st, B=2, H=3, Lq=5, Lk=5, D=64, dtype=1, table=d, td=0, b=bounds, n=3, off=0, out=d, ws=null,
            nb=0):
        return lib.wdit_rel_attention(q, qs, d, st, d, st, B, H, Lq, Lk, D, dtype, null, table, td, b, n, 1, 0, off,
                                      1.0, out, null, ws, nb, null)

    assert fwd(q=null) == 1 and fwd(qs=None) == 1 and fwd(table=null) == 1 and fwd(out=null) == 1 and fwd(b=None) == 1
    assert fwd(dtype=0) == 1 and fwd(td=3) == 1
    assert fwd(D=96) == 2 and fwd(H=0) == 2 and fwd(n=0) == 2 and fwd(off=-1) == 2 and fwd(Lk=0) == 2
    assert fwd(qs=zero) == 2 and fwd(qs=bad) == 3 and fwd(q=ctypes.c_void_p(0x1008)) == 3
    assert fwd(out=ctypes.c_void_p(0x1008)) == 3
    assert fwd(B=0, q=null, out=null) == 0 and fwd(Lq=0, q=null, out=null) == 0
    need = lib.wdit_rel_attention_workspace_bytes(1, 1, 1, 4096, 64)
    assert need > 0 and fwd(B=1, H=1, Lq=1, Lk=4096) == 5
    assert fwd(B=1, H=1, Lq=1, Lk=4096, ws=d, nb=need - 1) == 5
    assert lib.wdit_rel_attention_workspace_bytes(64, 64, 512, 512, 64) == 0

    def back(lse=d, dq=d, dt=d, ddt=0, ws=d, nb=1 << 30, Lq=5, Lk=5, gs=st):
        return lib.wdit_rel_attention_backward(d, st, d, st, d, st, d, gs, lse, 2, 3, Lq, Lk, 64, 1, null, d, 0,
                                               bounds, 3, 1, 0, 0, 1.0, dq, d, d, dt, ddt, ws, nb, null)

    assert back(lse=null) == 1 and back(dq=null) == 1 and back(dt=null) == 1
    assert back(ddt=-1) == 1
    assert back(Lq=0) == 2 and back(Lk=0) == 2 and back(gs=zero) == 2 and back(gs=bad) == 3
    assert back(dq=ctypes.c_void_p(0x1004)) == 3
    assert back(ws=null) == 5 and back(nb=16) == 5
