"""act(x W^T + bias) + residual and its gradients against the formulas in 64 bits.

Tolerances count roundings: half a step of the output's type, the fp32 sum (at most one step,
2^-23, per product added, of the sum of the products' sizes; |act'| <= 1.13), and 2^-16 of the
activation's value for its exponential (argument |z| <= 88: 88 * log2(e) * 2^-24 < 2^-16)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(autouse=True)
def _check_device_errors(pkg):
    yield
    pkg._lib.raise_on_device_error()


def act64(t, act):
    c0, c1 = math.sqrt(2 / math.pi), 0.044715
    return {"none": lambda: t, "relu": lambda: t.clamp_min(0), "silu": lambda: t / (1 + torch.exp(-t)),
            "gelu": lambda: 0.5 * t * torch.erfc(-t * math.sqrt(0.5)),
            "gelu_tanh": lambda: t / (1 + torch.exp(-2 * c0 * (t + c1 * t**3)))}[act]()


def dact64(t, act):
    t = t.detach().requires_grad_()
    with torch.enable_grad():
        (g,) = torch.autograd.grad(act64(t, act).sum(), t)
    return g


def make(m, n, k, dtype, bias=True, residual=True, seed=0, bias_dtype=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype).to(DEV)
    w = (torch.randn(n, k, generator=g) * k**-0.5).to(dtype).to(DEV)
    b = (0.5 * torch.randn(n, generator=g)).to(bias_dtype or dtype).to(DEV) if bias else None
    r = torch.randn(m, n, generator=g).to(dtype).to(DEV) if residual else None
    return x, w, b, r


def half(dtype):
    return torch.finfo(dtype).eps / 2


def check_forward(got, x, w, b, r, act):
    k = x.shape[1]
    pre = x.double() @ w.double().T
    size = x.double().abs() @ w.double().abs().T
    if b is not None:
        pre = pre + b.double()
        size = size + b.double().abs()
    y = act64(pre, act)
    want = y if r is None else y + r.double()
    sums = 1.13 * (k + 2) * 2.0**-23 * size
    tol = sums + 2.0**-16 * y.abs() + 1.01 * half(got.dtype) * want.abs() + torch.finfo(got.dtype).tiny
    tol = tol + half(got.dtype) * sums
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), (got.double() - want).abs().max().item())
    return pre


# rows / columns / reduction that reach every tile form: one row split over 8 CTAs, single tiles,
# two splits of rows, CTA pairs of both widths, ragged everything
SHAPES = [(1, 8, 8), (1, 1536, 8960), (1, 13824, 264), (2, 72, 4104), (3, 200, 72), (17, 64, 4096), (64, 4096, 1024),
          (127, 264, 136), (128, 512, 64), (129, 1536, 128), (300, 768, 1024), (513, 4608, 1536), (257, 264, 136),
          (1000, 1000, 520), (2049, 4104, 200)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forward_shapes(pkg, m, n, k, dtype):
    for i, act in enumerate(ACTS):
        x, w, b, r = make(m, n, k, dtype, bias=i != 1, residual=i != 2, seed=i)
        got = pkg.ops.linear_act_residual(x, w, b, act=act, residual=r)
        assert got.shape == (m, n) and got.dtype == dtype
        check_forward(got, x, w, b, r, act)


@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 40, 400])
def test_bias_types_and_unaligned_bias(pkg, m, bias_dtype):
    x, w, _, r = make(m, 264, 512, torch.bfloat16)
    b = torch.randn(300).to(bias_dtype).to(DEV)[3:267]
    check_forward(pkg.ops.linear_act_residual(x, w, b, act="silu", residual=r), x, w, b, r, "silu")


@pytest.mark.parametrize("m", [1, 5, 130, 600])
def test_views_leading_shapes_and_rows_behind(pkg, m):
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(m + 3, 600, generator=g).to(torch.bfloat16).to(DEV)
    for lo in (0, 8, 3):  # aligned rows, an aligned window, a window that has to be copied
        x = wide[1:m + 1, lo:lo + 520]
        _, w, b, r = make(m, 136, 520, torch.bfloat16)
        check_forward(pkg.ops.linear_act_residual(x, w, b, residual=r), x, w, b, r, "none")
        wv = torch.randn(136, 600, generator=g).to(torch.bfloat16).to(DEV)[:, lo:lo + 520]
        check_forward(pkg.ops.linear_act_residual(x, wv, b), x, wv, b, None, "none")
        wt = torch.randn(520, 136, generator=g).to(torch.bfloat16).to(DEV).T  # columns not contiguous
        check_forward(pkg.ops.linear_act_residual(x, wt, b), x, wt, b, None, "none")
    x, w, b, r = make(m, 136, 520, torch.bfloat16)
    y = pkg.ops.linear_act_residual(x.view(1, m, 520), w, b, residual=r.view(1, m, 136))
    assert y.shape == (1, m, 136) and torch.equal(y[0], pkg.ops.linear_act_residual(x, w, b, residual=r))
    y = pkg.ops.linear_act_residual(x[0], w, b, residual=r[0])
    check_forward(y[None], x[:1], w, b, r[:1], "none")
    # out=: writes its rows and nothing behind them; out may be the residual
    buf = torch.full((m + 2, 136), 7.0, dtype=torch.bfloat16, device=DEV)
    want = pkg.ops.linear_act_residual(x, w, b, act="gelu", residual=r)
    pkg.ops.linear_act_residual(x, w, b, act="gelu", residual=r, out=buf[:m])
    assert torch.equal(buf[:m], want) and (buf[m:] == 7).all()
    inplace = r.clone()
    assert pkg.ops.linear_act_residual(x, w, b, act="gelu", residual=inplace, out=inplace) is inplace
    assert torch.equal(inplace, want)


def test_no_rows(pkg):
    x, w, b, r = make(0, 64, 64, torch.bfloat16)
    assert pkg.ops.linear_act_residual(x, w, b, residual=r).shape == (0, 64)
    for t in (x, w, b, r):
        t.requires_grad_()
    out = pkg.ops.linear_act_residual(x, w, b, act="silu", residual=r)
    grads = torch.autograd.grad(out, [x, w, b, r], torch.zeros_like(out))
    assert grads[0].shape == (0, 64) and (grads[1] == 0).all() and (grads[2] == 0).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_infinite_and_nan_rows_stay_in_their_rows(pkg, act):
    x, w, b, r = make(200, 264, 128, torch.bfloat16)
    want = pkg.ops.linear_act_residual(x, w, b, act=act, residual=r)
    x[7] = float("nan")
    x[150, 3] = float("inf")
    got = pkg.ops.linear_act_residual(x, w, b, act=act, residual=r)
    keep = torch.ones(200, dtype=torch.bool)
    keep[[7, 150]] = False
    assert torch.equal(got[keep.to(DEV)], want[keep.to(DEV)])
    assert got[7].isnan().all()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_far_arguments(pkg, act):
    """Pre-activations far out: 0 or the value itself, no NaN (8 columns of weight +-1)."""
    x = torch.zeros(1, 8, dtype=torch.bfloat16, device=DEV)
    for v in (30.0, 100.0, 1e4, 1e30):
        x[0, 0] = v
        w = torch.zeros(8, 8, dtype=torch.bfloat16, device=DEV)
        w[0, 0], w[1, 0] = 1, -1
        xr = x.clone().requires_grad_()
        y = pkg.ops.linear_act_residual(xr, w, act=act)
        assert y[0, 0].item() == x[0, 0].item() and abs(y[0, 1].item()) < 1e-10
        (g,) = torch.autograd.grad(y, xr, torch.ones_like(y))
        assert g[0, 0].item() == 1.0


GRAD_SHAPES = [(1, 8, 8), (3, 72, 136), (64, 264, 520), (130, 512, 64), (513, 1000, 264), (2049, 264, 1536)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", GRAD_SHAPES)
def test_gradients(pkg, m, n, k, act, dtype):
    x, w, b, r = make(m, n, k, dtype, seed=11)
    dout = torch.randn(m, n, generator=torch.Generator().manual_seed(12)).to(dtype).to(DEV)
    for t in (x, w, b, r):
        t.requires_grad_()
    out = pkg.ops.linear_act_residual(x, w, b, act=act, residual=r)
    pre = check_forward(out.detach(), x.detach(), w.detach(), b.detach(), r.detach(), act)
    dx, dw, db, dr = torch.autograd.grad(out, [x, w, b, r], dout)
    assert torch.equal(dr, dout)
    x, w = x.detach().double(), w.detach().double()
    g, h = dout.double(), half(dtype)
    slope = dact64(pre, act) if act != "none" else torch.ones_like(pre)
    dpre = g * slope
    # pre is kept rounded (|act''| <= 1.2; for ReLU the sign of pre is safe outside its own error),
    # dpre is rounded before the products
    pre_err = h * pre.abs() + (k + 2) * 2.0**-23 * (x.abs() @ w.abs().T + b.detach().double().abs())
    if act == "none":
        err = torch.zeros_like(dpre)
    elif act == "relu":
        err = torch.where(pre.abs() <= pre_err, g.abs(), 0.0)
    else:
        err = g.abs() * (1.2 * pre_err + 2.0**-15)
    part = err + (0 if act == "none" else 1) * h * (dpre.abs() + err) + torch.finfo(dtype).tiny
    size = dpre.abs() + part
    tiny = torch.finfo(dtype).tiny

    def close(got, want, tol):
        tol = tol + 1.01 * h * (want.abs() + tol) + tiny
        bad = (got.double() - want).abs() > tol
        assert not bad.any(), (int(bad.sum()), ((got.double() - want).abs() / tol).max().item())

    close(dx, dpre @ w, part @ w.abs() + (n + 2) * 2.0**-23 * (size @ w.abs()))
    close(dw, dpre.T @ x, part.T @ x.abs() + (m + 2) * 2.0**-23 * (size.T @ x.abs()))
    close(db, dpre.sum(0), err.sum(0) + (m + 2) * 2.0**-24 * size.sum(0))


def test_gradient_against_differences(pkg):
    """fp32 differences of the op's own forward, sized so that the step dominates the rounding."""
    x, w, b, _ = make(40, 64, 48, torch.float16, residual=False, seed=21)
    weight = torch.randn(40, 64, device=DEV, dtype=torch.float64)
    w.requires_grad_()
    out = pkg.ops.linear_act_residual(x, w, b, act="gelu")
    (dw,) = torch.autograd.grad((out.double() * weight).sum().float(), w)
    d = torch.zeros_like(w)
    d[5, 7] = 0.25
    with torch.no_grad():
        hi = (pkg.ops.linear_act_residual(x, (w + d), b, act="gelu").double() * weight).sum()
        lo = (pkg.ops.linear_act_residual(x, (w - d), b, act="gelu").double() * weight).sum()
    step = ((w + d).double() - (w - d).double())[5, 7]
    diff = ((hi - lo) / step).item()
    # curvature: |act'''| <= 1.6, step 0.25 |x|; rounding: half a step of each changed output
    xs = x[:, 7].double().abs()
    curve = (weight[:, 5].abs() * 1.6 * xs**3).sum().item() * 0.25**2 / 6
    rounding = (weight[:, 5].abs() * (out[:, 5].double().abs() + 0.3 * xs)).sum().item() * 2.0**-11 * 2 / 0.5
    exact_err = 2.0**-10 * (weight[:, 5].abs() * xs).sum().item()
    assert abs(diff - dw[5, 7].item()) <= curve + rounding + exact_err


def test_only_the_gradients_asked_for(pkg):
    x, w, b, r = make(70, 64, 48, torch.bfloat16)
    full = [t.clone().requires_grad_() for t in (x, w, b, r)]
    dout = torch.randn(70, 64, device=DEV).to(torch.bfloat16)
    want = torch.autograd.grad(pkg.ops.linear_act_residual(full[0], full[1], full[2], act="silu", residual=full[3]),
                               full, dout)
    for i in range(4):
        ts = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b, r))]
        out = pkg.ops.linear_act_residual(ts[0], ts[1], ts[2], act="silu", residual=ts[3])
        (got,) = torch.autograd.grad(out, [ts[i]], dout)
        assert torch.equal(got, want[i])
    # a broadcast upstream gradient
    t = w.clone().requires_grad_()
    (got,) = torch.autograd.grad(pkg.ops.linear_act_residual(x, t, b, act="silu", residual=r).sum(), t)
    t2 = w.clone().requires_grad_()
    o2 = pkg.ops.linear_act_residual(x, t2, b, act="silu", residual=r)
    (want2,) = torch.autograd.grad(o2, t2, torch.ones_like(o2))
    assert torch.equal(got, want2)


def test_streams_and_graphs(pkg):
    x, w, b, r = make(48, 512, 1024, torch.bfloat16)
    want = pkg.ops.linear_act_residual(x, w, b, act="gelu", residual=r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = pkg.ops.linear_act_residual(x, w, b, act="gelu", residual=r)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    dout = torch.randn(48, 512, device=DEV).to(torch.bfloat16)

    def step():
        out = pkg.ops.linear_act_residual(leaves[0], leaves[1], leaves[2], act="gelu", residual=leaves[3])
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = [t.clone() for t in step()]
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, res in graphs:
        assert all(torch.equal(a, c) for a, c in zip(res, want))


def test_out_counts_as_written(pkg):
    """Autograd refuses a backward pass whose saved tensor out= has overwritten."""
    x = torch.randn(8, 64, device=DEV).to(torch.bfloat16)
    w = torch.randn(64, 64, device=DEV).to(torch.bfloat16).requires_grad_()
    h = torch.randn(8, 64, device=DEV).to(torch.bfloat16)
    y = pkg.ops.linear_act_residual(h, w)
    with torch.no_grad():
        pkg.ops.linear_act_residual(x, w, residual=h, out=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_rows_past_32_bit_offsets(pkg):
    g = torch.Generator().manual_seed(40)
    x = torch.randn(70, 128, generator=g).to(torch.bfloat16).to(DEV)
    w = torch.randn(64, 128, generator=g).to(torch.bfloat16).to(DEV)
    far = torch.empty(69 * (1 << 26) + 128, dtype=torch.bfloat16, device=DEV).as_strided((70, 128), (1 << 26, 1))
    far.copy_(x)
    assert torch.equal(pkg.ops.linear_act_residual(far, w, act="silu", residual=far[:, :64]),
                       pkg.ops.linear_act_residual(x, w, act="silu", residual=x[:, :64].contiguous()))


def test_gradients_of_more_row_chunks_than_a_grid_dimension_holds(pkg):
    """65536 chunks of 64 rows and five more rows; only some rows carry a gradient, so that the sums
    are exact in fp32 (small whole numbers) and every chunk boundary is met."""
    M = 65536 * 64 + 5
    x = torch.ones(M, 8, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(8, 8, dtype=torch.bfloat16, device=DEV)
    b = torch.ones(8, device=DEV)
    xs, ws, bs = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    dout = torch.zeros(M, 8, dtype=torch.bfloat16, device=DEV)
    dout[::1_000_003] = 1.0
    dout[-1] = 2.0
    out = pkg.ops.linear_act_residual(xs, ws, bs, act="relu")  # pre = 1: act' = 1
    dx, dw, db = torch.autograd.grad(out, [xs, ws, bs], dout)
    total = dout.float().sum(0)
    assert torch.equal(out, torch.ones_like(out)) and not dx.any()
    assert torch.equal(db, total) and torch.equal(dw.float(), total[:, None].expand(8, 8))


def test_one_row_without_a_batch_dimension(pkg):
    g = torch.Generator().manual_seed(41)
    x, w, r = (torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV) for s in ((64,), (32, 64), (32,)))
    want = pkg.ops.linear_act_residual(x[None], w, act="relu", residual=r[None])[0]
    assert torch.equal(pkg.ops.linear_act_residual(x, w, act="relu", residual=r), want)
    ts = [t.clone().requires_grad_() for t in (x, w, r)]
    out = pkg.ops.linear_act_residual(ts[0], ts[1], act="relu", residual=ts[2])
    out.sum().backward()  # a broadcast gradient
    assert out.shape == (32,) and all(t.grad.shape == t.shape for t in ts) and (ts[2].grad == 1).all()


def test_the_same_tensor_as_operand_and_residual(pkg):
    g = torch.Generator().manual_seed(42)
    x, w = (torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV) for s in ((40, 64), (64, 64)))
    assert torch.equal(pkg.ops.linear_act_residual(x, w, residual=x), pkg.ops.linear_act_residual(x, w, residual=x.clone()))
    with pytest.raises(ValueError, match="overlaps an operand"):
        pkg.ops.linear_act_residual(x, w, out=x)
