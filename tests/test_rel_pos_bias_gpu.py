"""Relative position bias by buckets and its gradient, against the rule in 64 bits."""
import functools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U32 = 2.0**-24  # half a step of fp32


@pytest.fixture(autouse=True)
def _check_device_errors(pkg):
    yield
    pkg._lib.raise_on_device_error()


@functools.lru_cache(maxsize=None)
def bucket(d, num_buckets, max_distance, bidirectional):
    """The rule, one relative position at a time, in whole numbers."""
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


def bucket_map(lq, lk, off, num_buckets, max_distance, bidirectional):
    line = torch.tensor([bucket(d, num_buckets, max_distance, bidirectional) for d in range(-(lq - 1) - off, lk - off)])
    i = torch.arange(lq)[:, None]
    return line[torch.arange(lk)[None, :] - i + lq - 1].to(DEV)


CASES = [
    # lq, lk, off, buckets, max_distance, bidirectional
    (1, 1, 0, 32, 128, True),
    (1, 4097, 4096, 32, 128, False),
    (7, 13, 0, 8, 5, True),
    (33, 31, 2, 32, 128, True),
    (128, 256, 0, 32, 128, True),
    (129, 257, 128, 32, 128, False),
    (300, 520, 0, 64, 500, True),
    (40, 2056, 1000, 16, 100, True),
    (65, 4100, 17, 2, 3, False),
    (5, 70, 0, 512, 1000, True),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lq,lk,off,nb,md,bi", CASES)
def test_bias_is_the_table_by_bucket(pkg, lq, lk, off, nb, md, bi, dtype):
    H = 3
    table = torch.randn(nb, H, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    got = pkg.ops.rel_pos_bias(table, lq, lk, bidirectional=bi, max_distance=md, q_offset=off)
    want = table[bucket_map(lq, lk, off, nb, md, bi)].permute(2, 0, 1)
    assert got.dtype == dtype and got.is_contiguous()
    assert torch.equal(got, want)  # a copy: no rounding


def test_bias_keeps_infinities_and_nan_of_the_table(pkg):
    table = torch.randn(32, 2, device=DEV)
    table[3, 0], table[20, 1], table[0, 1] = -float("inf"), float("nan"), torch.finfo(torch.float32).min
    got = pkg.ops.rel_pos_bias(table, 50, 60)
    want = table[bucket_map(50, 60, 0, 32, 128, True)].permute(2, 0, 1)
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("lq,lk,off,nb,md,bi", CASES)
def test_gradient_sums_cells_by_bucket(pkg, lq, lk, off, nb, md, bi, batch, dtype):
    H = 2
    g = torch.Generator().manual_seed(2)
    db = torch.randn(batch, H, lq, lk, generator=g).to(dtype).to(DEV)
    got = pkg.ops.rel_pos_bias_grad(db, nb, bidirectional=bi, max_distance=md, q_offset=off)
    where = bucket_map(lq, lk, off, nb, md, bi).flatten()
    want = torch.zeros(nb, H, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(want)
    for h in range(H):
        want[:, h].index_add_(0, where, db[:, h].double().sum(0).flatten())
        size[:, h].index_add_(0, where, db[:, h].double().abs().sum(0).flatten())
    assert got.shape == (nb, H) and got.dtype == torch.float32
    # A cell passes through at most 128 adds down its diagonal, 5 across lanes, 13 pieces for each
    # of the (at most 3 * 3 * 17) strips of a warp, 8 warps and the partial buckets (<= 16 here).
    adds = 128 + 5 + 13 * 153 + 8 + 16
    assert ((got.double() - want).abs() <= adds * U32 * size).all()
    again = pkg.ops.rel_pos_bias_grad(db, nb, bidirectional=bi, max_distance=md, q_offset=off)
    assert torch.equal(got, again)


@pytest.mark.parametrize("make", [
    lambda g: torch.randn(2, 3, 70, 90, generator=g).to(DEV)[:, :, 1:60, 3:80],       # unaligned window
    lambda g: torch.randn(2, 70, 3, 96, generator=g).to(DEV).transpose(1, 2),         # heads inside rows
    lambda g: torch.randn(2, 3, 96, 70, generator=g).to(DEV).transpose(2, 3),         # columns not contiguous
    lambda g: torch.randn(1, 3, 1, 96, generator=g).to(DEV).expand(2, 3, 40, 96),     # broadcast
    lambda g: torch.randn(3, 40, 96, generator=g).to(torch.bfloat16).to(DEV)[:, :, 8:],
])
def test_gradient_takes_views(pkg, make):
    db = make(torch.Generator().manual_seed(3))
    got = pkg.ops.rel_pos_bias_grad(db, 32)
    want = pkg.ops.rel_pos_bias_grad(db.contiguous().clone(), 32)
    size = db.double().abs().sum()
    assert ((got - want).abs() <= 2 * 1024 * U32 * size).all()  # the two may add in another order


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradient_is_rounded_once_to_the_type_asked_for(pkg, dtype):
    db = torch.randn(2, 3, 70, 90, generator=torch.Generator().manual_seed(5)).to(DEV)
    got = pkg.ops.rel_pos_bias_grad(db, 32, dtype=dtype)
    assert got.dtype == dtype
    assert torch.equal(got, pkg.ops.rel_pos_bias_grad(db, 32).to(dtype))
    none = pkg.ops.rel_pos_bias_grad(db[:, :, :0], 32, dtype=dtype)
    assert none.dtype == dtype and none.shape == (32, 3) and not none.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_table_that_starts_at_any_element(pkg, dtype):
    table = torch.randn(32, 3, generator=torch.Generator().manual_seed(6)).to(dtype).to(DEV)
    odd = torch.empty(32 * 3 + 1, dtype=dtype, device=DEV)[1:].view(32, 3).copy_(table)
    assert torch.equal(pkg.ops.rel_pos_bias(odd, 40, 50), pkg.ops.rel_pos_bias(table, 40, 50))


def test_more_row_tiles_than_a_grid_dimension_holds(pkg):
    lq = 65536 * 32 + 5
    table = torch.randn(32, 1, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(DEV)
    got = pkg.ops.rel_pos_bias(table, lq, 3, q_offset=1)
    for i0 in (0, 100, 65535 * 32 - 180, lq - 200):  # 200 rows each
        where = bucket_map(200, 3, 1 + i0, 32, 128, True)
        assert torch.equal(got[:, i0 : i0 + 200], table[where].permute(2, 0, 1))
    db = torch.zeros(1, lq, 3, device=DEV)
    db[0, ::100_000, 1] = 1.0
    want = torch.zeros(32, 1, device=DEV)
    for i in range(0, lq, 100_000):
        want[bucket(max(1 - (i + 1), -200), 32, 128, True)] += 1.0
    assert torch.equal(pkg.ops.rel_pos_bias_grad(db, 32, q_offset=1), want)


def test_gradient_cells_past_32_bit_offsets(pkg):
    db = torch.randn(70, 90, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).to(DEV)
    far = torch.empty(69 * (1 << 26) + 90, dtype=torch.bfloat16, device=DEV).as_strided((1, 70, 90), (0, 1 << 26, 1))
    far[0].copy_(db)
    assert torch.equal(pkg.ops.rel_pos_bias_grad(far, 32), pkg.ops.rel_pos_bias_grad(db[None].contiguous(), 32))


def test_gradient_of_no_cells_is_zero(pkg):
    for shape in [(0, 2, 5, 6), (2, 2, 0, 6), (2, 2, 5, 0)]:
        got = pkg.ops.rel_pos_bias_grad(torch.empty(shape, device=DEV), 32)
        assert got.shape == (32, 2) and (got == 0).all()
    assert pkg.ops.rel_pos_bias(torch.ones(32, 2, device=DEV), 0, 7).shape == (2, 0, 7)
    assert pkg.ops.rel_pos_bias(torch.ones(32, 2, device=DEV), 7, 0).shape == (2, 7, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd_and_differences(pkg, dtype):
    g = torch.Generator().manual_seed(4)
    table = torch.randn(32, 3, generator=g).to(dtype).to(DEV).requires_grad_()
    weight = torch.randn(2, 3, 40, 50, generator=g).to(dtype).to(DEV)
    bias = pkg.ops.rel_pos_bias(table, 40, 50)
    (bias[None] * weight).sum().backward()
    want = pkg.ops.rel_pos_bias_grad(weight.float().sum(0).to(dtype), 32).to(dtype)
    assert table.grad.dtype == dtype and torch.equal(table.grad, want)
    # linear in the table: a difference of any step is the gradient
    step = torch.zeros_like(table)
    step[5, 1] = 1.0
    with torch.no_grad():
        cells = pkg.ops.rel_pos_bias(step, 40, 50).double() * weight.double().sum(0)
    size = cells.abs().sum().item()
    assert abs(cells.sum().item() - table.grad[5, 1].item()) <= 4 * torch.finfo(dtype).eps * size + 1024 * U32 * size


def test_other_stream_and_captured_graph(pkg):
    table = torch.randn(32, 4, device=DEV)
    db = torch.randn(1, 4, 64, 72, device=DEV)
    want_b, want_g = pkg.ops.rel_pos_bias(table, 64, 72), pkg.ops.rel_pos_bias_grad(db, 32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got_b, got_g = pkg.ops.rel_pos_bias(table, 64, 72), pkg.ops.rel_pos_bias_grad(db, 32)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got_b, want_b) and torch.equal(got_g, want_g)
    graphs = []
    for _ in range(2):  # two graphs: each has its own workspace
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = (pkg.ops.rel_pos_bias(table, 64, 72), pkg.ops.rel_pos_bias_grad(db, 32))
        graphs.append((gr, out))
    table.mul_(2)
    db.mul_(-1)
    for gr, _ in graphs:
        gr.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out[0], 2 * want_b) and torch.equal(out[1], -want_g)
