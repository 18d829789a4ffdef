"""The text-encoder operators in a run, as a text encoder's layer and a decoder's cached step use them.

layer: qkv = x Wqkv^T; a = rel_pos_attention(q, k, v, table); h = a Wo^T + x;
       y = gelu_tanh(h W1^T + b1) W2^T + b2 + h

The exact values are the layer in 64 bits. The tolerance is what the rounding of the stored tensors
does on its own: the same layer in 64 bits with every tensor that the operators hand on in 16 bits
rounded there (forward: qkv, P, a, h, pre-activation, f, y; backward: their gradients and dS). Both
errors are sums of the same number of roundings of thousands of cells, so their norms agree up to a
few per cent; the operators may be off by twice that norm.
fp32 sums are far below these roundings wherever a result is not 0. The table's gradient can be: with
one key dS = P (dP - delta) is 0, and what is left of it are the fp32 sums of dP and delta, each at
most (D + 2) 2^-23 sum |da v| off; that is added to its tolerance, over all its cells."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, D, C, F = 4, 64, 192, 512
BUCKETS, FAR = 32, 128


@pytest.fixture(autouse=True)
def _check_device_errors(pkg):
    yield
    pkg._lib.raise_on_device_error()


def parameters(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def r(*shape, std, dt=dtype):
        return (torch.randn(*shape, generator=g) * std).to(dt).to(DEV)

    return dict(wqkv=r(3 * H * D, C, std=C**-0.5), wo=r(C, H * D, std=(H * D) ** -0.5), table=r(BUCKETS, H, std=1.0),
                w1=r(F, C, std=C**-0.5), b1=r(F, std=0.3, dt=torch.float32), w2=r(C, F, std=F**-0.5),
                b2=r(C, std=0.3, dt=torch.float32))


def layer(ops, p, x, k_lens):
    B, L, _ = x.shape
    q, k, v = ops.linear_act_residual(x, p["wqkv"]).view(B, L, 3, H, D).unbind(2)
    a = ops.rel_pos_attention(q, k, v, p["table"], k_lens=k_lens, scale=0.125, max_distance=FAR)
    h = ops.linear_act_residual(a.reshape(B, L, H * D), p["wo"], residual=x)
    f = ops.linear_act_residual(h, p["w1"], p["b1"], act="gelu_tanh")
    return ops.linear_act_residual(f, p["w2"], p["b2"], residual=h)


class Rounded(torch.autograd.Function):
    """A 64-bit tensor as its 16-bit copy holds it, and its gradient too."""

    @staticmethod
    def forward(ctx, t, dtype, forward, backward):
        ctx.dtype = dtype if backward else None
        return t.to(dtype).double() if forward else t.clone()

    @staticmethod
    def backward(ctx, g):
        return (g if ctx.dtype is None else g.to(ctx.dtype).double()), None, None, None


def plain(pkg, p, x, k_lens, dtype=None, keep=None):
    """The layer in 64 bits; dtype: with the operators' roundings."""
    def r(t, forward=True, backward=True):
        return t if dtype is None else Rounded.apply(t, dtype, forward, backward)

    B, L, _ = x.shape
    q, k, v = r(x @ p["wqkv"].T).view(B, L, 3, H, D).permute(2, 0, 3, 1, 4).unbind(0)
    bounds = torch.tensor(pkg.ops.rel_pos_bounds(BUCKETS, FAR, True), device=DEV)
    i = torch.arange(L, device=DEV)
    d = i[None, :] - i[:, None]
    where = torch.searchsorted(bounds, d.abs(), right=True) + (d > 0) * (BUCKETS // 2)
    z = r(0.125 * (q @ k.transpose(-1, -2)) + p["table"][where].permute(2, 0, 1), forward=False)
    z = z.masked_fill((i[None, :] >= k_lens[:, None])[:, None, None], -torch.inf)
    pr = r(torch.softmax(z, -1), backward=False)
    o = r(pr @ v)
    if keep is not None:
        o.retain_grad()
        keep.update(o=o, pr=pr, v=v)
    a = o.transpose(1, 2).reshape(B, L, H * D)
    h = r(a @ p["wo"].T + x)
    pre = r(h @ p["w1"].T + p["b1"], forward=False)
    f = r(torch.nn.functional.gelu(pre, approximate="tanh"))
    return r(f @ p["w2"].T + p["b2"] + h)


def gradients(run, p, x, dout, convert):
    leaves = {n: convert(t).requires_grad_() for n, t in {**p, "x": x}.items()}
    out = run({n: t for n, t in leaves.items() if n != "x"}, leaves["x"])
    out.backward(convert(dout))
    return {"out": out.detach(), **{"d" + n: t.grad for n, t in leaves.items()}}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L", [1, 77, 300])
def test_layer_and_its_gradients(pkg, L, dtype):
    g = torch.Generator().manual_seed(50)
    p, B = parameters(dtype), 3
    x, dout = (torch.randn(B, L, C, generator=g).to(dtype).to(DEV) for _ in range(2))
    lens = torch.tensor([L, max(1, L // 3), max(1, L - 1)], dtype=torch.int32, device=DEV)
    wide = lambda t: t.detach().double()  # noqa: E731
    keep = {}
    exact = gradients(lambda p, x: plain(pkg, p, x, lens, keep=keep), p, x, dout, wide)
    sums = (keep["pr"].detach() * (keep["o"].grad.abs() @ keep["v"].detach().abs().transpose(-1, -2))).sum((0, 2, 3))  # per head
    fp32 = {"dtable": (2 * (D + 2) * 2.0**-23 * sums).norm()}
    rounded = gradients(lambda p, x: plain(pkg, p, x, lens, dtype), p, x, dout, wide)
    got = gradients(lambda p, x: layer(pkg.ops, p, x, lens), p, x, dout, lambda t: t.detach().clone())
    for n, e in exact.items():
        h = torch.finfo(got[n].dtype).eps / 2  # the result's own rounding
        allowed = 2 * ((rounded[n] - e).norm() + h * e.norm()) + fp32.get(n, 0.0)
        assert got[n].isfinite().all() and (got[n].double() - e).norm() <= allowed, n


def test_layer_in_a_graph(pkg):
    p, L = parameters(torch.bfloat16), 200
    g = torch.Generator().manual_seed(51)
    x, dout, x2, dout2 = (torch.randn(2, L, C, generator=g).to(torch.bfloat16).to(DEV) for _ in range(4))
    lens = torch.tensor([L, 50], dtype=torch.int32, device=DEV)
    leaves = {n: t.requires_grad_() for n, t in p.items()}
    sx, sd = x.clone().requires_grad_(), dout.clone()

    def step():
        out = layer(pkg.ops, leaves, sx, lens)
        return [out.detach(), *torch.autograd.grad(out, [sx, *leaves.values()], sd)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for xs, ds, ln in ((x, dout, [L, 50]), (x2, dout2, [0, L]), (x2, dout, [3, 130])):
        with torch.no_grad():
            sx.copy_(xs), sd.copy_(ds), lens.copy_(torch.tensor(ln, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in res]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_cached_steps_agree_with_the_whole(pkg):
    """One token at a time over a cache against one causal call: the same products, other tiles and
    key splits, so a result differs by the rounding of both (half a step each) and of P (half a step
    of each weight, and fp32 sums below that)."""
    dtype, L = torch.bfloat16, 150
    h = torch.finfo(dtype).eps / 2
    g = torch.Generator().manual_seed(52)
    q, k, v = (torch.randn(2, L, H, D, generator=g).to(dtype).to(DEV) for _ in range(3))
    table = torch.randn(BUCKETS, H, generator=g).to(DEV)
    kw = dict(bidirectional=False, max_distance=FAR)
    whole = pkg.ops.rel_pos_attention(q, k, v, table, causal=True, **kw).double()
    cache_k, cache_v = (torch.full((2, 256, H, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    bound = pkg.ops.rel_pos_attention(q, k, v.abs(), table, causal=True, **kw).double()  # sum P |v|
    for n in range(L):
        cache_k[:, n], cache_v[:, n] = k[:, n], v[:, n]
        lens = torch.full((2,), n + 1, dtype=torch.int32, device=DEV)
        one = pkg.ops.rel_pos_attention(q[:, n : n + 1], cache_k, cache_v, table, k_lens=lens, q_offset=n, **kw)
        tol = 2 * h * whole[:, n : n + 1].abs() + 3 * h * bound[:, n : n + 1]
        assert ((one.double() - whole[:, n : n + 1]).abs() <= tol).all(), n


def test_layers_on_two_streams_at_once(pkg):
    """Enough CTAs of every kernel that both streams' share the SMs and their tensor memory."""
    L, B = 300, 40
    g = torch.Generator().manual_seed(53)
    p = [{n: t.requires_grad_() for n, t in parameters(torch.bfloat16, seed=s).items()} for s in (1, 2)]
    xs = [torch.randn(B, L, C, generator=g).to(torch.bfloat16).to(DEV).requires_grad_() for _ in range(2)]
    dout = torch.randn(B, L, C, generator=g).to(torch.bfloat16).to(DEV)
    lens = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32).to(DEV)

    def step(i):
        out = layer(pkg.ops, p[i], xs[i], lens)
        return [out.detach(), *torch.autograd.grad(out, [xs[i], *p[i].values()], dout)]

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append((i, step(i)))
    torch.cuda.synchronize()
    for i, res in got:
        assert all(torch.equal(a, b) for a, b in zip(res, want[i]))
