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


def probabilities(pkg, q, k, table, *, scale=None, causal=False, bidirectional=True, max_distance=128, q_offset=0):
    """P in 64 bits and the error that 32-bit scores leave in it, relative (see below)."""
    B, Lq, H, D = q.shape
    Lk, scale = k.shape[1], D**-0.5 if scale is None else scale
    q, k = (t.double().transpose(1, 2) for t in (q, k))
    bias = table.double().T[:, buckets(pkg, Lq, Lk, table.shape[0], max_distance, bidirectional, q_offset)][None]
    z = scale * (q @ k.transpose(-1, -2)) + bias
    seen = torch.ones(Lq, Lk, dtype=torch.bool, device=DEV)
    if causal:
        seen = torch.arange(Lk, device=DEV)[None] <= torch.arange(Lq, device=DEV)[:, None] + q_offset
    z = torch.where(seen, z, -torch.inf)
    # a score: D fp32 adds of exact products, scaling, bias, maximum (and its power of two): a step each
    size = abs(scale) * (q.abs() @ k.abs().transpose(-1, -2)) + bias.abs() + z.amax(-1, keepdim=True).abs() + 28
    dz = (D + 4) * 2.0**-23 * torch.where(seen, size, 0.0)
    return torch.softmax(z, -1), 2 * dz.amax(-1, keepdim=True) + 2.0**-20


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
