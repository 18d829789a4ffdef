"""act(x W^T + bias) + residual where its arithmetic ends: every value of the types through each activation
and its derivative."""
import math

import pytest
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
