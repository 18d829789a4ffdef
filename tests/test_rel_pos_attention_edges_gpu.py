"""Attention with the relative position bias where its arithmetic ends: keys that nobody sees, values
and biases at the ends of their types, small gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _check_device_errors(pkg):
    yield
    pkg._lib.raise_on_device_error()


def make(B, H, Lq, Lk, D, dtype, nb=32, seed=0):
    g = torch.Generator().manual_seed(seed)

    def r(*s, dt=dtype):
        return torch.randn(*s, generator=g).to(dt).to(DEV)

    return r(B, Lq, H, D), r(B, Lk, H, D), r(B, Lk, H, D), r(nb, H, dt=torch.float32), r(B, Lq, H, D)


def out_and_gradients(pkg, q, k, v, table, dout, **kw):
    ts = [t.detach().clone().requires_grad_() for t in (q, k, v, table)]
    out = pkg.ops.rel_pos_attention(*ts, **kw)
    return [out.detach(), *torch.autograd.grad(out, ts, dout)]


def buckets(pkg, lq, lk, nb, md, bi, off):
    bounds = torch.tensor(pkg.ops.rel_pos_bounds(nb, md, bi), device=DEV)
    d = torch.arange(lk, device=DEV)[None] - torch.arange(lq, device=DEV)[:, None] - off
    n = d.abs() if bi else (-d).clamp_min(0)
    return torch.searchsorted(bounds, n, right=True) + (d > 0) * (nb // 2 if bi else 0)


def probabilities(pkg, q, k, table, *, scale=None, causal=False, bidirectional=True, max_distance=128, q_offset=0,
                  k_lens=None):
    """P in 64 bits and the error that 32-bit scores leave in it, relative (see below)."""
    B, Lq, H, D = q.shape
    Lk, scale = k.shape[1], D**-0.5 if scale is None else scale
    q, k = (t.double().transpose(1, 2) for t in (q, k))
    bias = table.double().T[:, buckets(pkg, Lq, Lk, table.shape[0], max_distance, bidirectional, q_offset)][None]
    z = scale * (q @ k.transpose(-1, -2)) + bias
    seen = torch.ones(Lq, Lk, dtype=torch.bool, device=DEV)
    if causal:
        seen = torch.arange(Lk, device=DEV)[None] <= torch.arange(Lq, device=DEV)[:, None] + q_offset
    if k_lens is not None:
        seen = seen & (torch.arange(Lk, device=DEV)[None] < k_lens[:, None])[:, None, None]
    z = torch.where(seen, z, -torch.inf)
    # a score: D fp32 adds of exact products, scaling, bias, maximum (and its power of two): a step each
    top = z.amax(-1, keepdim=True)
    size = abs(scale) * (q.abs() @ k.abs().transpose(-1, -2)) + bias.abs() + top.abs() + 28
    dz = (D + 4) * 2.0**-23 * torch.where(seen, size, 0.0)
    p = torch.where(top == -torch.inf, 0.0, torch.softmax(z, -1))  # a row without keys
    return p, 2 * dz.amax(-1, keepdim=True) + 2.0**-20


def within(got, want, tol):
    """(NaN is never within.)"""
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), ((got.double() - want).abs() / tol).nan_to_num(torch.inf).max().item())


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("B,H,Lq,Lk,D", [(1, 2, 1, 1, 64), (1, 2, 70, 64, 128), (2, 2, 1, 3000, 128), (1, 3, 200, 1100, 64),
                                         (8, 40, 129, 300, 64)])
def test_bf16_values_near_the_largest_and_the_smallest(pkg, B, H, Lq, Lk, D, rising):
    """O is a mean of v: finite however large v, and whatever a later score adds to the first ones. Small
    values keep their precision (down to 2^-80 here)."""
    q, k, v, table, _ = make(B, H, Lq, Lk, D, torch.bfloat16, seed=2)
    if rising:  # scores rise by about 2^60 over the keys
        k = (k * torch.linspace(0.02, 12, Lk, device=DEV)[None, :, None, None]).to(torch.bfloat16)
    p, eps = probabilities(pkg, q, k, table)
    h = 2.0**-8  # half a step of bf16
    for power in (126, 100, 0, -80):
        # |v| in [0.5, 2) 2^power
        vs = (torch.sign(v.float()) * (0.5 + 1.49 * torch.sigmoid(v.float())) * 2.0**power).to(torch.bfloat16)
        got = pkg.ops.rel_pos_attention(q, k, vs, table)
        x = vs.double().transpose(1, 2)
        want, mean = p @ x, p @ x.abs()
        tol = mean * (h + eps + (Lk + 2) * 2.0**-23)  # P to 16 bits, scores, sums
        within(got, want.transpose(1, 2), (tol + 1.01 * h * (want.abs() + tol)).transpose(1, 2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H,Lq,Lk,off", [
    (1, 2, 1, 300, 0),        # a token whose cache holds itself only
    (2, 2, 1, 3000, 1234),    # ... keys split over CTAs, the last one inside a tile
    (2, 3, 37, 200, 90),      # a chunk of a prompt
    (1, 2, 200, 500, 0),      # two query tiles; a cache that is longer than what was written
    (8, 40, 129, 400, 64),    # more CTAs than two per SM
])
def test_keys_past_the_last_query_may_hold_anything(pkg, B, H, Lq, Lk, off, D, dtype):
    q, k, v, table, dout = make(B, H, Lq, Lk, D, dtype, seed=1)
    kw = dict(causal=True, bidirectional=False, q_offset=off)
    want = out_and_gradients(pkg, q, k, v, table, dout, **kw)
    assert all(t.isfinite().all() for t in want)
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
        k2, v2 = k.clone(), v.clone()
        k2[:, off + Lq:], v2[:, off + Lq:] = bad, bad
        assert torch.equal(pkg.ops.rel_pos_attention(q, k2, v2, table, **kw), want[0])
        got = out_and_gradients(pkg, q, k2, v2, table, dout, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not want[2][:, off + Lq:].any() and not want[3][:, off + Lq:].any()


MASKS = [(torch.float32, torch.finfo(torch.float32).min), (torch.float32, -1e9), (torch.float32, -1e30),
         (torch.bfloat16, torch.finfo(torch.bfloat16).min), (torch.float16, torch.finfo(torch.float16).min)]


@pytest.mark.parametrize("table_dtype,mask", MASKS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Lq,Lk,D", [(1, 2, 200, 200, 64), (2, 3, 130, 270, 128), (1, 2, 2, 3000, 64),
                                         (8, 40, 129, 129, 64)])
def test_masks_of_the_lowest_value(pkg, B, H, Lq, Lk, D, dtype, table_dtype, mask):
    """Head 0: keys ahead of the query are masked. Head 1: all keys; what is left are their scores. The
    oracle's mask is -20000, which 64 bits tell scores apart beside."""
    q, k, v, table, dout = make(B, H, Lq, Lk, D, dtype, seed=3)
    table[16:], table[:, 1] = mask, mask
    table = table.to(table_dtype)
    masked = table.double() <= -60000
    p, _ = probabilities(pkg, q, k, torch.where(masked, -20000.0, table.double()))
    # errors of P: as in probabilities() for the scores, with the biases that are no masks; where only
    # masks are seen, maximum and log-sum are rounded at 2^14 (2^-10 each, twice with split keys)
    _, eps = probabilities(pkg, q, k, torch.where(masked, 0.0, table.double()))
    eps = eps + 2.0**-8 * torch.ones(H, device=DEV, dtype=torch.float64).index_fill(
        0, torch.tensor([h for h in range(H) if h != 1], device=DEV), 0.0)[None, :, None, None]
    h = torch.finfo(dtype).eps / 2
    sub = 2.0**-25 if dtype == torch.float16 else 0.0
    got = out_and_gradients(pkg, q, k, v, table, dout)
    assert all(t.isfinite().all() for t in got)
    x, do = v.double().transpose(1, 2), dout.double().transpose(1, 2)
    want = p @ x
    tol = (p @ x.abs()) * (h + eps + (Lk + 2) * 2.0**-23) + sub * x.abs().sum(-2, keepdim=True)
    tol = tol + 1.01 * h * (want.abs() + tol) + torch.finfo(dtype).tiny
    within(got[0], want.transpose(1, 2), tol.transpose(1, 2))
    # dv = P^T dO with P to 16 bits
    want = p.transpose(-1, -2) @ do
    tol = (p * (eps + h) + sub + Lq * 2.0**-23 * p).transpose(-1, -2) @ do.abs()
    tol = tol + 1.01 * h * (want.abs() + tol) + torch.finfo(dtype).tiny
    within(got[3], want.transpose(1, 2), tol.transpose(1, 2))
    # dq = scale dS k, dS = P (dP - delta): dP and delta are fp32 sums of D and Lk terms
    dp = do @ x.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_dp = (D + 2) * 2.0**-23 * (do.abs() @ x.abs().transpose(-1, -2))
    e_delta = (p * ((eps + (Lk + 2) * 2.0**-23) * dp.abs() + e_dp)).sum(-1, keepdim=True)
    e_ds = p * (eps * (dp - delta).abs() + e_dp + e_delta) * (1 + h) + h * ds.abs() + sub
    kk, scale = k.double().transpose(1, 2), D**-0.5
    want = scale * (ds @ kk)
    tol = scale * ((e_ds + Lk * 2.0**-23 * ds.abs()) @ kk.abs())
    tol = tol + 1.01 * h * (want.abs() + tol) + torch.finfo(dtype).tiny
    within(got[1], want.transpose(1, 2), tol.transpose(1, 2))


def test_masks_of_minus_infinity_hide_and_nan_stays(pkg):
    q, k, v, table, dout = make(1, 2, 70, 90, 64, torch.float16, seed=4)
    table[:, 0] = -torch.inf
    table[3, 1] = torch.nan
    out = pkg.ops.rel_pos_attention(q, k, v, table)
    assert not out[:, :, 0].any() and out[:, 4:, 1].isnan().all() and out[:, :3, 1].isfinite().all()


def significand(t, bits):
    """Rounded to so many bits, at any exponent."""
    m, e = torch.frexp(t)
    return torch.ldexp(torch.round(m * 2.0**bits) * 2.0**-bits, e)


def gradients64(pkg, q, k, v, table, dout, *, bits=None, **kw):
    """dq, dk, dv in 64 bits; bits: P and dS rounded to that significand, at any exponent."""
    p, _ = probabilities(pkg, q, k, table, **kw)
    scale = kw.get("scale", q.shape[-1] ** -0.5)
    q, k, v, do = (t.double().transpose(1, 2) for t in (q, k, v, dout))
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    if bits is not None:
        p, ds = significand(p, bits), significand(ds, bits)
    res = scale * (ds @ k), scale * (ds.transpose(-1, -2) @ q), p.transpose(-1, -2) @ do
    return [t.transpose(1, 2) for t in res]


def as_good_as_rounding(pkg, got, q, k, v, table, dout, **kw):
    """fp16 gradients may be off by twice what rounding P and dS to its 11 bits (without the ends of its
    range) and then the results to fp16 gives; errors are sums of thousands of independent roundings,
    so their norms agree to a few per cent. fp32 sums lie far below."""
    exact = gradients64(pkg, q, k, v, table, dout, **kw)
    rounded = gradients64(pkg, q, k, v, table, dout, bits=11, **kw)
    for name, g, e, r in zip(("dq", "dk", "dv"), got, exact, rounded):
        allowed = 2 * (r.to(torch.float16).double() - e).norm()
        assert g.isfinite().all() and e.norm() > 0, name
        assert (g.double() - e).norm() <= allowed, (name, ((g.double() - e).norm() / e.norm()).item(),
                                                   (allowed / e.norm()).item())


@pytest.mark.parametrize("std", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("B,H,Lq,Lk,D,kw", [
    (1, 2, 512, 2048, 64, {}), (1, 2, 300, 4096, 128, {}), (2, 3, 257, 333, 64, dict(causal=True, q_offset=40)),
    (1, 1, 3000, 77, 128, {}), (1, 2, 1, 1000, 64, {})])
def test_fp16_gradients_of_any_loss_scale(pkg, B, H, Lq, Lk, D, kw, std):
    q, k, v, table, dout = make(B, H, Lq, Lk, D, torch.float16, seed=5)
    dout = (dout.float() * std).to(torch.float16)
    got = out_and_gradients(pkg, q, k, v, table, dout, **kw)
    as_good_as_rounding(pkg, got[1:4], q, k, v, table, dout, **kw)


def test_fp16_gradients_of_rows_of_different_sizes(pkg):
    """Each row's dq has its own factor."""
    q, k, v, table, dout = make(1, 2, 300, 1500, 64, torch.float16, seed=6)
    size = torch.tensor([1.0, 1e-3, 1e-4], device=DEV).repeat(100)
    dout = (dout.float() * size[None, :, None, None]).to(torch.float16)
    got = out_and_gradients(pkg, q, k, v, table, dout)
    as_good_as_rounding(pkg, got[1:4], q, k, v, table, dout)
    exact, rounded = (gradients64(pkg, q, k, v, table, dout, bits=b)[0] for b in (None, 11))
    for n in range(3):
        e = exact[:, n::3]
        assert (got[1][:, n::3].double() - e).norm() <= 2 * (rounded[:, n::3].to(torch.float16).double() - e).norm(), n


def test_fp16_gradients_of_many_flat_keys(pkg):
    """P is 2^-16 here, below fp16's normal numbers."""
    q, k, v, table, dout = make(1, 1, 70, 1 << 16, 64, torch.float16, seed=7)
    got = out_and_gradients(pkg, q, k, v, table, dout, scale=0.03)
    as_good_as_rounding(pkg, got[1:4], q, k, v, table, dout, scale=0.03)


def test_fp16_gradients_whose_score_gradients_pass_the_type(pkg):
    """dS reaches 10^6, dq, dk and dv do not."""
    q, k, v, table, dout = make(1, 2, 100, 90, 64, torch.float16, seed=8)
    q, k, v, dout = ((t.float() * f).to(torch.float16) for t, f in ((q, 2.0**-9), (k, 2.0**-9), (v, 200), (dout, 200)))
    p, _ = probabilities(pkg, q, k, table * 3)
    dp = dout.double().transpose(1, 2) @ v.double().permute(0, 2, 3, 1)
    assert (p * (dp - (p * dp).sum(-1, keepdim=True))).abs().max() > 65504
    got = out_and_gradients(pkg, q, k, v, table * 3, dout)
    as_good_as_rounding(pkg, got[1:4], q, k, v, table * 3, dout)


def test_fp16_gradients_beside_a_row_without_a_number(pkg):
    """An infinity in one query's gradient reaches what that query touches and nothing else."""
    q, k, v, table, dout = make(2, 2, 130, 150, 64, torch.float16, seed=9)
    want = out_and_gradients(pkg, q, k, v, table, dout)
    dout = dout.clone()
    dout[1, 7, 0, 3] = torch.inf
    got = out_and_gradients(pkg, q, k, v, table, dout)
    keep = torch.ones(2, 130, 2, dtype=torch.bool, device=DEV)
    keep[1, 7, 0] = False
    assert torch.equal(got[1][keep], want[1][keep])
    for n in (2, 3):
        assert torch.equal(got[n][0], want[n][0]) and torch.equal(got[n][1, :, 1], want[n][1, :, 1])
    assert torch.equal(got[4][:, 1], want[4][:, 1])


def test_fp16_gradients_of_nothing_are_zero(pkg):
    q, k, v, table, dout = make(1, 2, 70, 90, 64, torch.float16, seed=10)
    got = out_and_gradients(pkg, q, k, v, table, torch.zeros_like(dout))
    assert not any(t.any() for t in got[1:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [dict(), dict(lens=True), dict(causal=True, bidirectional=False), dict(causal=True, lens=True)])
@pytest.mark.parametrize("B,H,Lq,Lk,D", [(2, 3, 5, 7, 128), (3, 2, 129, 257, 64), (1, 2, 64, 1000, 128), (3, 3, 640, 65, 64),
                                         (3, 3, 900, 2, 64), (3, 3, 900, 5, 128), (2, 3, 1500, 280, 64)])
def test_gradients_with_delta_from_fp32_sums(pkg, B, H, Lq, Lk, D, kw, dtype):
    """delta = rowsum(P dP) is an fp32 sum of what dS is made of, not of the rounded output: no cell of dS, and
    no bucket of the table, whose cells cancel, carries half a step of a 16-bit type of |dO| |out|."""
    q, k, v, table, dout = make(B, H, Lq, Lk, D, dtype, seed=11)
    kw = dict(kw, q_offset=max(0, Lk - Lq) if "causal" in kw else 0)
    if kw.pop("lens", False):
        kw["k_lens"] = torch.tensor([Lk, max(1, Lk // 2), 0][:B], dtype=torch.int32, device=DEV)
    got = out_and_gradients(pkg, q, k, v, table, dout, **kw)
    p, eps = probabilities(pkg, q, k, table, **kw)
    where = buckets(pkg, Lq, Lk, 32, 128, kw.get("bidirectional", True), kw["q_offset"]).flatten()
    U, h, scale = 2.0**-23, torch.finfo(dtype).eps / 2, D**-0.5
    q, k, v, do = (t.double().transpose(1, 2) for t in (q, k, v, dout))
    dp = do @ v.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_dp = (D + 2) * U * (do.abs() @ v.abs().transpose(-1, -2))
    e_delta = (p * ((eps + (Lk + 2) * U) * dp.abs() + e_dp)).sum(-1, keepdim=True)
    e_ds = p * (eps * (dp - delta).abs() + e_dp + e_delta)
    # operands of 16 bits: half a step, and in fp16 2^-38 of the bound that dS was taken up to 2^14 by
    # (2^-39 of P, which is at most 1)
    cell, cell_k, cell_p = h * (ds.abs() + e_ds), 0.0, 0.0
    if dtype == torch.float16:
        bound = (p * dp.abs()).amax(-1, keepdim=True) + delta.abs()
        cell, cell_k, cell_p = cell + 1.1 * 2.0**-38 * bound, 1.1 * 2.0**-38 * bound.amax(-2, keepdim=True), 2.0**-39
    tiny = torch.finfo(dtype).smallest_normal * h

    def near(got, want, tol):
        within(got, want.transpose(1, 2), (tol + 1.01 * h * (want.abs() + tol) + tiny).transpose(1, 2))

    near(got[1], scale * (ds @ k), scale * ((e_ds + cell + Lk * U * ds.abs()) @ k.abs()))
    near(got[2], scale * (ds.transpose(-1, -2) @ q),
         scale * ((e_ds + cell + cell_k + Lq * U * ds.abs()).transpose(-1, -2) @ q.abs()))
    near(got[3], p.transpose(-1, -2) @ do, (p * (eps + h + Lq * U) + cell_p).transpose(-1, -2) @ do.abs())
    depth = 32 + 16 + 5 + 2 * (Lk // 32 + 2) + 8 + B * (Lq // 128 + 1)  # adds a cell of the table's sums passes
    for head in range(H):
        want, tol = (torch.zeros(32, dtype=torch.float64, device=DEV) for _ in range(2))
        want.index_add_(0, where, ds[:, head].sum(0).flatten())
        tol.index_add_(0, where, (e_ds + depth * U * (ds.abs() + e_ds))[:, head].sum(0).flatten())
        within(got[4][:, head], want, tol + 2.0**-24 * want.abs() + 1e-30)


@pytest.mark.parametrize("nb,md,bi", [(512, 1000, True), (512, 257, True), (256, 256, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tables_that_fill_shared_memory(pkg, nb, md, bi, dtype):
    """The largest lines and sums of head size 128: gradients against those of a bias tensor."""
    q, k, v, table, dout = make(1, 2, 150, 400, 128, dtype, nb=nb, seed=12)
    kw = dict(max_distance=md, bidirectional=bi, q_offset=30)
    got = out_and_gradients(pkg, q, k, v, table, dout, **kw)
    assert all(t.isfinite().all() for t in got)
    exact = gradients64(pkg, q, k, v, table, dout, **kw)
    rounded = gradients64(pkg, q, k, v, table, dout, bits=11 if dtype == torch.float16 else 8, **kw)
    for g, e, r in zip(got[1:4], exact, rounded):
        assert (g.double() - e).norm() <= 2 * (r.to(dtype).double() - e).norm()


def test_fp16_gradients_in_graphs_and_on_two_streams(pkg):
    """The bounds of dS lie in the call's own workspace."""
    sets = [make(2, 3, 200, 300, 64, torch.float16, seed=20 + i) for i in range(2)]
    sets = [(*s[:4], (s[4].float() * 10.0 ** (-2 * i)).to(torch.float16)) for i, s in enumerate(sets)]
    lens = torch.tensor([300, 111], dtype=torch.int32, device=DEV)
    leaves = [[t.requires_grad_() for t in s[:4]] for s in sets]

    def step(i):
        out = pkg.ops.rel_pos_attention(*leaves[i], k_lens=lens)
        return [out.detach(), *torch.autograd.grad(out, leaves[i], sets[i][4])]

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(i)
        graphs.append((g, res))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i][0].replay()
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append((i, step(i)))
    torch.cuda.synchronize()
    for i, res in [*enumerate(g[1] for g in graphs), *got]:
        assert all(torch.equal(a, b) for a, b in zip(res, want[i]))
