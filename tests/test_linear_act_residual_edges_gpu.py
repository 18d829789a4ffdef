"""act(x W^T + bias) + residual where its arithmetic ends: every value of the types through each activation
and its derivative."""
import math

import pytest
import test_linear_act_residual_gpu as base
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _check_device_errors(pkg):
    yield
    pkg._lib.raise_on_device_error()


def every_value(dtype):
    t = torch.arange(65536, dtype=torch.int32, device=DEV).to(torch.int16).view(dtype)
    t = t[t.isfinite()]
    return t.view(-1, 8)


def within(got, want, tol):
    """(NaN is never within.)"""
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), ((got.double() - want).abs() / tol).nan_to_num(torch.inf).max().item())


def formulas(x, act):
    """act, act' and the sum of the sizes of act's derivative's terms, in 64 bits."""
    if act == "none":
        return x, torch.ones_like(x), torch.ones_like(x)
    if act == "relu":
        return x.clamp_min(0), (x > 0).double(), (x > 0).double()
    if act == "gelu":
        cdf, pdf = 0.5 * torch.erfc(-x * math.sqrt(0.5)), torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
        pdf = torch.where(pdf == 0, 0.0, x * pdf)
        return x * cdf, cdf + pdf, cdf + pdf.abs()
    if act == "silu":
        z, dz = x, torch.ones_like(x)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        z, dz = c * (x + 0.044715 * x**3), c * (1 + 3 * 0.044715 * x * x)
    s = torch.sigmoid(z)
    slope = s * torch.sigmoid(-z)
    slope = torch.where(slope == 0, 0.0, x * slope * dz)
    return x * s, s + slope, s + slope.abs()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("size", [1.0, 2.0**10])
def test_every_value_through_the_activation_and_its_derivative(pkg, act, dtype, size):
    """An identity weight: the pre-activation is x itself, dx is dpre. Errors: half a step of the type; 2^-15 of
    the value's terms (the exponential of an argument of up to 88 that has been rounded three times,
    88 * 3 * 2^-24, and what it enters); what lies below 2^-126 in between may be 0."""
    x = every_value(dtype).requires_grad_()
    w = torch.eye(8, dtype=dtype, device=DEV)
    out = pkg.ops.linear_act_residual(x, w, act=act)
    (dx,) = torch.autograd.grad(out, x, torch.full_like(out, size))
    y, slope, terms = formulas(x.detach().double(), act)
    h = torch.finfo(dtype).eps / 2
    below = torch.finfo(dtype).smallest_normal * h  # half a step of the smallest numbers
    within(out.detach(), y, (h + 2.0**-15) * y.abs() + below + 2.0**-119)  # x to 2^7 there
    keep = slope * size < torch.finfo(dtype).max
    within(dx[keep], (slope * size)[keep], (h * slope.abs() * size + 2.0**-15 * terms * size + below + size * 2.0**-119)[keep])


# The comparisons of test_linear_act_residual_gpu.py ask for an error above the tolerance, which NaN never
# is: the same calls, cell by cell a number.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", base.SHAPES)
def test_every_form_gives_numbers(pkg, m, n, k, dtype):
    for i, act in enumerate(base.ACTS):
        x, w, b, r = base.make(m, n, k, dtype, bias=i != 1, residual=i != 2, seed=i)
        assert pkg.ops.linear_act_residual(x, w, b, act=act, residual=r).isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", base.ACTS)
@pytest.mark.parametrize("m,n,k", base.GRAD_SHAPES)
def test_gradients_are_numbers(pkg, m, n, k, act, dtype):
    ts = [t.requires_grad_() for t in base.make(m, n, k, dtype, seed=11)]
    dout = torch.randn(m, n, generator=torch.Generator().manual_seed(12)).to(dtype).to(DEV)
    out = pkg.ops.linear_act_residual(ts[0], ts[1], ts[2], act=act, residual=ts[3])
    assert all(t.isfinite().all() for t in (out.detach(), *torch.autograd.grad(out, ts, dout)))


@pytest.mark.parametrize("m", [1, 40, 400])
def test_views_and_bias_types_give_numbers(pkg, m):
    for bias_dtype in (torch.float32, torch.bfloat16, torch.float16):
        x, w, _, r = base.make(m, 264, 512, torch.bfloat16)
        b = torch.randn(300).to(bias_dtype).to(DEV)[3:267]
        assert pkg.ops.linear_act_residual(x, w, b, act="silu", residual=r).isfinite().all()
    wide = torch.randn(m + 3, 600).to(torch.bfloat16).to(DEV)
    for lo in (0, 8, 3):
        _, w, b, r = base.make(m, 136, 520, torch.bfloat16)
        assert pkg.ops.linear_act_residual(wide[1:m + 1, lo:lo + 520], w, b, residual=r).isfinite().all()


@pytest.mark.parametrize("m,n,k", [(1, 1536, 8960), (300, 768, 1024), (513, 4608, 1536), (2049, 4104, 200)])
def test_no_cell_is_left_unwritten(pkg, m, n, k):
    """out= filled with NaN first, in every tile form; nothing behind it is touched."""
    x, w, b, r = base.make(m, n, k, torch.bfloat16)
    room = torch.full((m * n + 1024,), torch.nan, dtype=torch.bfloat16, device=DEV)
    out = room[:m * n].view(m, n)
    pkg.ops.linear_act_residual(x, w, b, act="gelu", residual=r, out=out)
    assert out.isfinite().all() and room[m * n:].isnan().all()
    base.check_forward(out, x, w, b, r, "gelu")
