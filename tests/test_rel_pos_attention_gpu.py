"""Attention with the bias read from its table, and its gradients, against the formulas in 64 bits.

The tolerances follow the arithmetic, cell by cell. h = half a step of the 16-bit type.
  score      the fp32 sum of D exact products (a step, 2^-23, each), its scaling, the bias and the
             subtraction of the maximum: dz <= (D + 4) 2^-23 (scale sum|q k| + |bias| + |max|)
  P          relative error eps = 2 dz + 2^-20 (exponential, row sum), then h when it becomes an
             operand (fp16: at least 2^-25, below its normal numbers)
  out        sum P |v| (eps + h + Lk 2^-23), then h |out|
  dS         P (eps |dP - delta| + d(dP) + d(delta)); delta is formed from the rounded out
  dq, dk, dv sums of the above against the other operand, then h of the result
  dtable     the sum of the errors of dS, fp32 sums"""
import functools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-23


@pytest.fixture(autouse=True)
def _check_device_errors(pkg):
    yield
    pkg._lib.raise_on_device_error()


@functools.lru_cache(maxsize=None)
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


def bucket_map(lq, lk, off, nb, md, bi):
    clip = md + 1
    line = torch.tensor([bucket(max(-clip, min(clip, d)), nb, md, bi) for d in range(-(lq - 1) - off, lk - off)])
    i = torch.arange(lq)[:, None]
    return line[torch.arange(lk)[None, :] - i + lq - 1].to(DEV)


def make(B, H, Lq, Lk, D, dtype, nb=32, seed=0, table_dtype=torch.float32, q_std=1.0):
    g = torch.Generator().manual_seed(seed)

    def r(*s, std=1.0, dt=dtype):
        return (torch.randn(*s, generator=g) * std).to(dt).to(DEV)

    return r(B, Lq, H, D, std=q_std), r(B, Lk, H, D), r(B, Lk, H, D), r(nb, H, dt=table_dtype)


def check(got, q, k, v, table, *, k_lens=None, scale=None, causal=False, bidirectional=True, max_distance=128,
          q_offset=0, dout=None):
    """got: out, or (out, dq, dk, dv, dtable) with dout."""
    B, Lq, H, D = q.shape
    Lk = k.shape[1]
    scale = D**-0.5 if scale is None else scale
    h = torch.finfo(q.dtype).eps / 2
    sub = 2.0**-25 if q.dtype == torch.float16 else 0.0
    tiny = torch.finfo(q.dtype).smallest_normal
    lens = torch.full((B,), Lk) if k_lens is None else k_lens.cpu().clamp(0, Lk)
    where = bucket_map(Lq, Lk, q_offset, table.shape[0], max_distance, bidirectional)
    j = torch.arange(Lk, device=DEV)
    seen = (j[None, :] < lens.to(DEV)[:, None])[:, None, None, :].expand(B, 1, Lq, Lk)
    if causal:
        seen = seen & (j[None, :] <= torch.arange(Lq, device=DEV)[:, None] + q_offset)
    live = (j[None, :] < lens.to(DEV)[:, None])[:, :, None, None]
    q, k, v = q.double().transpose(1, 2), k.double(), v.double()
    k = torch.where(live, k, 0.0).transpose(1, 2)  # what lies behind a sample's keys is not looked at
    v = torch.where(live, v, 0.0).transpose(1, 2)
    bias = table.double().T[:, where][None]
    z = scale * (q @ k.transpose(-1, -2)) + bias
    z = torch.where(seen, z, -torch.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -torch.inf, 0.0, top)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    finite_bias = torch.where(bias.isfinite(), bias.abs(), 0.0)
    dz = (D + 4) * U * (abs(scale) * (q.abs() @ k.abs().transpose(-1, -2)) + finite_bias + top.abs())
    eps = 2 * torch.where(seen, dz, 0.0).amax(-1, keepdim=True) + 2.0**-20
    o = p @ v
    out_tol = (p @ v.abs()) * (h + eps + (Lk + 2) * U) + sub * (v.abs().sum(-2, keepdim=True))
    out_tol = out_tol + 1.01 * h * (o.abs() + out_tol) + tiny

    def close(name, g, want, tol):
        g = g.double().transpose(1, 2) if g.dim() == 4 else g.double()
        bad = ~((g - want).abs() <= tol)
        assert not bad.any(), (name, int(bad.sum()), ((g - want).abs() / tol).max().item())

    if dout is None:
        close("out", got, o, out_tol)
        return
    close("out", got[0], o, out_tol)
    do = dout.double().transpose(1, 2)
    dp = do @ v.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_dp = (D + 2) * U * (do.abs() @ v.abs().transpose(-1, -2))
    e_delta = (do.abs() * out_tol).sum(-1, keepdim=True) + (D + 2) * U * (do * o).abs().sum(-1, keepdim=True)
    e_ds = p * (eps * (dp - delta).abs() + e_dp + e_delta)
    r_ds = e_ds + h * (ds.abs() + e_ds) + sub * seen
    r_p = p * (eps + h) + sub * seen

    def fin(want, tol):
        return tol + 1.01 * h * (want.abs() + tol) + tiny

    dv = p.transpose(-1, -2) @ do
    dq = scale * (ds @ k)
    dk = scale * (ds.transpose(-1, -2) @ q)
    close("dv", got[3], dv, fin(dv, r_p.transpose(-1, -2) @ do.abs() + Lq * U * (p.transpose(-1, -2) @ do.abs())))
    close("dq", got[1], dq, fin(dq, abs(scale) * (r_ds @ k.abs() + Lk * U * (ds.abs() @ k.abs()))))
    close("dk", got[2], dk, fin(dk, abs(scale) * (r_ds.transpose(-1, -2) @ q.abs()
                                                  + Lq * U * (ds.abs().transpose(-1, -2) @ q.abs()))))
    nb = table.shape[0]
    want, tol = (torch.zeros(nb, H, dtype=torch.float64, device=DEV) for _ in range(2))
    cells = where.flatten()
    depth = 32 + 16 + 5 + 2 * (Lk // 32 + 2) + 8 + B * (Lq // 128 + 1)  # adds a cell passes through
    for hh in range(H):
        want[:, hh].index_add_(0, cells, ds[:, hh].sum(0).flatten())
        tol[:, hh].index_add_(0, cells, (e_ds + depth * U * (ds.abs() + e_ds))[:, hh].sum(0).flatten())
    ht = torch.finfo(table.dtype).eps / 2
    close("dtable", got[4], want, tol + 1.01 * ht * (want.abs() + tol) + 1e-30)


SHAPES = [(1, 1, 1, 1, 64), (2, 3, 5, 7, 128), (1, 2, 128, 128, 64), (3, 2, 129, 257, 64), (2, 1, 300, 300, 128),
          (1, 2, 64, 1000, 128), (2, 2, 1, 2100, 64), (1, 1, 200, 2500, 128), (1, 3, 640, 65, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Lq,Lk,D", SHAPES)
def test_forward(pkg, B, H, Lq, Lk, D, dtype):
    for n, (causal, bi, off) in enumerate([(False, True, 0), (True, False, max(0, Lk - Lq)), (False, False, 3)]):
        q, k, v, table = make(B, H, Lq, Lk, D, dtype, seed=n)
        lens = torch.tensor([Lk, Lk // 2, 1][:B], dtype=torch.int32, device=DEV) if n != 1 else None
        kw = dict(k_lens=lens, causal=causal, bidirectional=bi, q_offset=off)
        got = pkg.ops.rel_pos_attention(q, k, v, table, **kw)
        assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous()
        check(got, q, k, v, table, **kw)


@pytest.mark.parametrize("nb,md,bi", [(32, 128, True), (2, 2, False), (512, 3000, True), (8, 5, True), (64, 70, False)])
@pytest.mark.parametrize("table_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_bucket_rules_and_table_types(pkg, nb, md, bi, table_dtype):
    q, k, v, table = make(1, 2, 200, 330, 64, torch.bfloat16, nb=nb, seed=3, table_dtype=table_dtype)
    kw = dict(bidirectional=bi, max_distance=md, q_offset=40, scale=0.07)
    check(pkg.ops.rel_pos_attention(q, k, v, table, **kw), q, k, v, table, **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Lq", [1, 100])
def test_lengths_and_what_lies_behind_them(pkg, Lq, D):
    lens = [0, 1, 63, 64, 65, 128, 700, 999, 1000, -5, 2000]
    B, Lk = len(lens), 1000
    q, k, v, table = make(B, 2, Lq, Lk, D, torch.bfloat16, seed=4)
    kl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = pkg.ops.rel_pos_attention(q, k, v, table, k_lens=kl)
    check(want, q, k, v, table, k_lens=kl)
    for bad in (float("nan"), float("inf"), torch.finfo(torch.bfloat16).min):
        k2, v2 = k.clone(), v.clone()
        for b, n in enumerate(lens):
            k2[b, max(n, 0):], v2[b, max(n, 0):] = bad, bad
        assert torch.equal(pkg.ops.rel_pos_attention(q, k2, v2, table, k_lens=kl), want)
    assert (want[0] == 0).all() and (want[9] == 0).all()


@pytest.mark.parametrize("make_view", [
    lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),              # [B, H, L, D] in memory
    lambda t: torch.cat([t, t, t], -1).contiguous()[..., t.shape[-1]:2 * t.shape[-1]],  # packed heads
    lambda t: torch.cat([t, t], 1)[:, : t.shape[1]],                        # rows behind the last one
    lambda t: torch.nn.functional.pad(t, (3, 5))[..., 3:-5],               # unaligned: copied
    lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2),          # D not contiguous: copied
])
def test_layouts(pkg, make_view):
    q, k, v, table = make(2, 3, 150, 170, 64, torch.float16, seed=5)
    want = pkg.ops.rel_pos_attention(q, k, v, table)
    got = pkg.ops.rel_pos_attention(make_view(q), make_view(k), make_view(v), table)
    assert torch.equal(got, want)
    one = k[:1, :, :1].expand(2, 170, 3, 64)  # broadcast samples and heads: strides of 0
    check(pkg.ops.rel_pos_attention(q, one, v, table), q, one.contiguous(), v, table)


def test_large_scores_and_masked_buckets(pkg):
    """Scores far apart (the running maximum moves), a bucket of -inf, rows it leaves empty."""
    q, k, v, table = make(1, 2, 260, 700, 64, torch.bfloat16, seed=6)
    k = (k * torch.linspace(0.1, 12, 700, device=DEV)[None, :, None, None]).to(torch.bfloat16)
    check(pkg.ops.rel_pos_attention(q, k, v, table, scale=0.5), q, k, v, table, scale=0.5)
    k = k.flip(1).contiguous()
    check(pkg.ops.rel_pos_attention(q, k, v, table, scale=0.5), q, k, v, table, scale=0.5)
    table[16:] = -torch.inf  # every key ahead of the query
    table[0, 1] = -torch.inf  # head 1: itself too
    got = pkg.ops.rel_pos_attention(q, k, v, table)
    check(got, q, k, v, table)
    assert (got[0, 0, 1] == 0).all() and not got.isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Lq,Lk", [(5, 31, 300, 300), (3, 110, 130, 77), (330, 1, 1, 500), (2, 100, 257, 1)])
def test_more_ctas_than_two_per_sm(pkg, B, H, Lq, Lk, dtype):
    q, k, v, table = make(B, H, Lq, Lk, 64, dtype, seed=16)
    k = (k * torch.linspace(0.1, 12, Lk, device=DEV)[None, :, None, None]).to(dtype)  # the maximum moves
    lens = torch.tensor([[Lk, 0, Lk // 2, 65, 64][b % 5] for b in range(B)], dtype=torch.int32, device=DEV)
    for kw in (dict(k_lens=lens), dict(causal=True, bidirectional=False, q_offset=max(0, Lk - Lq)),
               dict(k_lens=lens, causal=True, q_offset=7, scale=0.4)):
        want = pkg.ops.rel_pos_attention(q, k, v, table, **kw)
        check(want, q, k, v, table, **kw)
        if "k_lens" in kw:
            behind = (torch.arange(Lk, device=DEV)[None] >= lens[:, None])[..., None, None]
            k2, v2 = k.masked_fill(behind, float("nan")), v.masked_fill(behind, float("inf"))
            assert torch.equal(pkg.ops.rel_pos_attention(q, k2, v2, table, **kw), want)


def test_flat_scores(pkg):
    q, k, v, table = make(1, 1, 64, 3000, 128, torch.float16, seed=7)
    q.zero_(), table.zero_()
    check(pkg.ops.rel_pos_attention(q, k, v, table), q, k, v, table)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Lq,Lk,D", SHAPES)
def test_gradients(pkg, B, H, Lq, Lk, D, dtype):
    for n, (causal, bi, off) in enumerate([(False, True, 0), (True, False, max(0, Lk - Lq)), (True, True, 5)]):
        q, k, v, table = (t.requires_grad_() for t in make(B, H, Lq, Lk, D, dtype, seed=n))
        lens = torch.tensor([Lk, 0, 1][:B], dtype=torch.int32, device=DEV) if n == 0 else None
        kw = dict(k_lens=lens, causal=causal, bidirectional=bi, q_offset=off, scale=None if n else 0.11)
        dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(9)).to(dtype).to(DEV)
        out = pkg.ops.rel_pos_attention(q, k, v, table, **kw)
        grads = torch.autograd.grad(out, [q, k, v, table], dout)
        check((out.detach(), *grads), *(t.detach() for t in (q, k, v, table)), dout=dout, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Lq,Lk", [(3, 110, 130, 77), (5, 31, 300, 300)])
def test_gradients_of_more_ctas_than_two_per_sm(pkg, B, H, Lq, Lk, dtype):
    q, k, v, table = (t.requires_grad_() for t in make(B, H, Lq, Lk, 64, dtype, seed=21))
    lens = torch.tensor([[Lk, 0, Lk // 2, 65, 64][b % 5] for b in range(B)], dtype=torch.int32, device=DEV)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(22)).to(dtype).to(DEV)
    for kw in (dict(k_lens=lens), dict(causal=True, q_offset=5)):
        out = pkg.ops.rel_pos_attention(q, k, v, table, **kw)
        grads = torch.autograd.grad(out, [q, k, v, table], dout)
        check((out.detach(), *grads), *(t.detach() for t in (q, k, v, table)), dout=dout, **kw)


def test_gradients_of_some_inputs_and_a_summed_output(pkg):
    """Only what is asked for is returned; the gradient of a sum arrives as a broadcast tensor; the
    same tensor as q, k and v gets the sum of the three."""
    q, k, v, table = make(2, 2, 70, 70, 64, torch.bfloat16, seed=23)
    ones = torch.ones_like(q)
    ts = [t.clone().requires_grad_() for t in (q, k, v, table)]
    want = torch.autograd.grad(pkg.ops.rel_pos_attention(*ts), ts, ones)
    for n in range(4):
        args = [t.clone() for t in (q, k, v, table)]
        args[n].requires_grad_()
        pkg.ops.rel_pos_attention(*args).sum().backward()
        assert torch.equal(args[n].grad, want[n])
    x = q.clone().requires_grad_()
    (got,) = torch.autograd.grad(pkg.ops.rel_pos_attention(x, x, x, table), x, ones)
    three = [q.clone().requires_grad_() for _ in range(3)]
    parts = torch.autograd.grad(pkg.ops.rel_pos_attention(*three, table), three, ones)
    total = sum(p.double() for p in parts)
    step = 2.0**-8 * sum(p.double().abs() for p in parts)  # two rounded adds, half a step each
    assert ((got.double() - total).abs() <= 2 * step).all()


@pytest.mark.parametrize("nb,md,bi", [(2, 2, False), (512, 3000, True), (8, 5, True), (64, 70, False)])
def test_gradients_of_bucket_rules(pkg, nb, md, bi):
    q, k, v, table = (t.requires_grad_() for t in make(2, 2, 200, 330, 64, torch.bfloat16, nb=nb, seed=3))
    kw = dict(bidirectional=bi, max_distance=md, q_offset=40)
    out = pkg.ops.rel_pos_attention(q, k, v, table, **kw)
    dout = torch.randn_like(out)
    grads = torch.autograd.grad(out, [q, k, v, table], dout)
    check((out.detach(), *grads), *(t.detach() for t in (q, k, v, table)), dout=dout, **kw)


@pytest.mark.parametrize("D", [64, 128])
def test_gradients_ignore_what_lies_behind(pkg, D):
    lens = [0, 1, 64, 100, 257, 300]
    q, k, v, table = make(len(lens), 2, 140, 300, D, torch.bfloat16, seed=8)
    kl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    dout = torch.randn_like(q)

    def grads(k, v):
        ts = [t.clone().requires_grad_() for t in (q, k, v, table)]
        out = pkg.ops.rel_pos_attention(*ts, k_lens=kl)
        return [out.detach(), *torch.autograd.grad(out, ts, dout)]

    want = grads(k, v)
    check(want, q, k, v, table, k_lens=kl, dout=dout)
    k2, v2 = k.clone(), v.clone()
    for b, n in enumerate(lens):
        k2[b, n:], v2[b, n:] = float("nan"), float("inf")
    got = grads(k2, v2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for b, n in enumerate(lens):
        assert (got[2][b, n:] == 0).all() and (got[3][b, n:] == 0).all()


def test_masked_buckets_have_finite_gradients(pkg):
    q, k, v, table = make(1, 2, 200, 200, 64, torch.bfloat16, seed=10)
    table[16:] = -torch.inf
    table[0, 1] = -torch.inf
    ts = [t.requires_grad_() for t in (q, k, v, table)]
    out = pkg.ops.rel_pos_attention(*ts)
    dout = torch.randn_like(out)
    grads = torch.autograd.grad(out, ts, dout)
    check((out.detach(), *grads), *(t.detach() for t in ts), dout=dout)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Lq,Lk", [(900, 1), (900, 2), (900, 5), (300, 64), (300, 65), (200, 200), (200, 256),
                                   (2000, 280), (130, 1100)])
def test_table_gradient_of_few_keys(pkg, Lq, Lk, D):
    """Most rows' cells fall into one bucket there, where their sum is 0: what is left of it are fp32
    errors, not half steps of a 16-bit type. Per cell P (eps |dP - delta| + d(dP) + d(delta)), delta
    the fp32 sum of P dP over the row; then the sums of the table."""
    B, H, nb = 2, 3, 32
    q, k, v, table = make(B, H, Lq, Lk, D, torch.bfloat16, seed=18)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(19)).to(torch.bfloat16).to(DEV)
    t = table.clone().requires_grad_()
    (got,) = torch.autograd.grad(pkg.ops.rel_pos_attention(q, k, v, t), t, dout)
    where = bucket_map(Lq, Lk, 0, nb, 128, True)
    q, k, v, do = (x.double().transpose(1, 2) for x in (q, k, v, dout))
    bias = table.double().T[:, where][None]
    z = D**-0.5 * (q @ k.transpose(-1, -2)) + bias
    p, dp = torch.softmax(z, -1), do @ v.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dz = (D + 4) * U * (D**-0.5 * (q.abs() @ k.abs().transpose(-1, -2)) + bias.abs() + z.amax(-1, keepdim=True).abs())
    eps = 2 * dz.amax(-1, keepdim=True) + 2.0**-20
    e_dp = (D + 2) * U * (do.abs() @ v.abs().transpose(-1, -2))
    e_delta = (p * (eps * dp.abs() + e_dp)).sum(-1, keepdim=True) + (Lk + 2) * U * (p * dp.abs()).sum(-1, keepdim=True)
    e_ds = p * (eps * (dp - delta).abs() + e_dp + e_delta)
    depth = 32 + 16 + 5 + 2 * (Lk // 32 + 2) + 8 + B * (Lq // 128 + 1)
    for h in range(H):
        want, tol = (torch.zeros(nb, dtype=torch.float64, device=DEV) for _ in range(2))
        want.index_add_(0, where.flatten(), ds[:, h].sum(0).flatten())
        tol.index_add_(0, where.flatten(), (e_ds + depth * U * (ds.abs() + e_ds))[:, h].sum(0).flatten())
        assert ((got[:, h].double() - want).abs() <= tol + 2.0**-24 * want.abs() + 1e-30).all()


def test_gradient_against_differences(pkg):
    """Central differences of the op's own forward along one direction per input."""
    q, k, v, table = make(1, 2, 70, 90, 64, torch.float16, seed=11)
    weight = torch.randn(1, 70, 2, 64, generator=torch.Generator().manual_seed(12)).to(torch.float16).to(DEV)
    ts = [t.clone().requires_grad_() for t in (q, k, v, table)]
    grads = torch.autograd.grad(pkg.ops.rel_pos_attention(*ts), ts, weight)
    for n, base in enumerate((q, k, v, table)):
        g = torch.Generator().manual_seed(20 + n)
        step = (torch.randint(0, 2, base.shape, generator=g) * 2 - 1).to(base.dtype).to(DEV) * 2.0**-5
        args = [q, k, v, table]
        res = []
        for s in (1, -1):
            args[n] = base + s * step
            res.append((pkg.ops.rel_pos_attention(*args).double() * weight.double()).sum().item())
        moved = ((base + step).double() - (base - step).double()) / 2
        want = (grads[n].double() * moved).sum().item()
        diff = (res[0] - res[1]) / 2
        # rounding of the two forwards (independent, half a step each: 8 standard deviations), the
        # gradients' own rounding, and the cubic term of a 2^-5 step (|d^3 out| bounded by the
        # spread of the scores it moves: 6 (sum |step| / 8)^3 is far below the first)
        outs = pkg.ops.rel_pos_attention(q, k, v, table).double()
        noise = 8 * 2.0**-11 * (outs * weight.double()).square().sum().sqrt().item() * 2
        own = 8 * 2.0**-10 * (grads[n].double() * moved).square().sum().sqrt().item()
        assert abs(diff - want) <= noise + own + 0.02 * abs(want), (n, diff, want, noise, own)


def test_repeats_bit_for_bit(pkg):
    q, k, v, table = make(2, 4, 500, 500, 64, torch.bfloat16, seed=13)
    ts = [t.requires_grad_() for t in (q, k, v, table)]
    dout = torch.randn_like(q)
    runs = []
    for _ in range(3):
        out = pkg.ops.rel_pos_attention(*ts)
        runs.append([out.detach(), *torch.autograd.grad(out, ts, dout)])
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_empty(pkg):
    for B, Lq, Lk in [(0, 4, 4), (2, 0, 4), (2, 4, 0)]:
        q, k, v, table = (t.requires_grad_() for t in make(B, 2, Lq, Lk, 64, torch.bfloat16))
        out = pkg.ops.rel_pos_attention(q, k, v, table)
        assert out.shape == (B, Lq, 2, 64) and (out == 0).all()
        grads = torch.autograd.grad(out, [q, k, v, table], torch.ones_like(out))
        assert all((g == 0).all() and g.shape == t.shape for g, t in zip(grads, (q, k, v, table)))


def test_streams_and_graphs(pkg):
    q, k, v, table = make(2, 2, 100, 900, 64, torch.bfloat16, seed=14)
    kl = torch.tensor([900, 300], dtype=torch.int32, device=DEV)
    want = pkg.ops.rel_pos_attention(q, k, v, table, k_lens=kl)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = pkg.ops.rel_pos_attention(q, k, v, table, k_lens=kl)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    ts = [t.clone().requires_grad_() for t in (q, k, v, table)]
    dout = torch.randn_like(q)

    def step():
        out = pkg.ops.rel_pos_attention(*ts, k_lens=kl)
        return [out.detach(), *torch.autograd.grad(out, ts, dout)]

    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    kl.copy_(torch.tensor([77, 900], dtype=torch.int32))  # lengths are read on the device
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = step()
    for _, res in graphs:
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_agrees_with_the_bias_tensor(pkg):
    """The bias tensor of rel_pos_bias in a plain masked softmax, and its gradient's path."""
    q, k, v, table = make(1, 4, 130, 150, 64, torch.float16, seed=15)
    t1, t2 = table.clone().requires_grad_(), table.clone().requires_grad_()
    dout = torch.randn_like(q)
    out = pkg.ops.rel_pos_attention(q, k, v, t1)
    (g1,) = torch.autograd.grad(out, t1, dout)
    bias = pkg.ops.rel_pos_bias(t2, 130, 150)
    z = (q.float().transpose(1, 2) @ k.float().permute(0, 2, 3, 1)) * 64**-0.5 + bias
    o2 = (torch.softmax(z, -1) @ v.float().transpose(1, 2)).transpose(1, 2)
    (g2,) = torch.autograd.grad(o2, t2, dout.float())
    assert (out.float() - o2).abs().max() <= 2.0**-9 * v.abs().max()
    assert (g1 - g2).norm() <= 2.0**-9 * g2.norm() + 2.0**-9


def test_cache_past_32_bit_offsets(pkg):
    """Rows of a cache 2^26 elements apart: the last ones lie behind 2^32 elements."""
    q, k, v, table = make(1, 2, 3, 70, 64, torch.bfloat16, seed=17)
    room = torch.empty(69 * (1 << 26) + 4 * 64, dtype=torch.bfloat16, device=DEV)
    fk, fv = (room[s:].as_strided((1, 70, 2, 64), (8, 1 << 26, 64, 1)) for s in (0, 128))
    fk.copy_(k), fv.copy_(v)
    kw = dict(causal=True, bidirectional=False, q_offset=67)
    dout = torch.randn_like(q)
    res = []
    for kk, vv in ((k, v), (fk, fv)):
        ts = [t.detach().requires_grad_() for t in (q, kk, vv, table)]
        out = pkg.ops.rel_pos_attention(*ts, **kw)
        res.append([out.detach(), *torch.autograd.grad(out, ts, dout)])
    assert all(torch.equal(a, b) for a, b in zip(*res))
    check(res[0], q, k, v, table, dout=dout, **kw)


def test_two_streams_at_once(pkg):
    """Calls that overlap on the device share nothing: key splits' workspaces, backward's partial sums."""
    sets = [make(2, 2, 9, 3000, 64, torch.bfloat16, seed=30 + i) for i in range(2)]
    dout = torch.randn_like(sets[0][0])

    def run(ts):
        ts = [t.detach().requires_grad_() for t in ts]
        out = pkg.ops.rel_pos_attention(*ts)
        return [out.detach(), *torch.autograd.grad(out, ts, dout)]

    want = [run(ts) for ts in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, ts in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(run(ts))
    torch.cuda.synchronize()
    for n, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[n % 2]))
