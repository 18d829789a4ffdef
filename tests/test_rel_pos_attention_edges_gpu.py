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
