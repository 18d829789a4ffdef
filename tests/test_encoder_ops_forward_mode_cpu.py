"""Forward-mode derivatives of the text-encoder operators are refused (fake tensors: CUDA ones without a
device)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode

BF = torch.bfloat16


def bias(ops, t):
    ops.rel_pos_bias(t[0], 4, 5)


def bias_grad(ops, t):
    ops.rel_pos_bias_grad(t[0], 32)


def attention(ops, t):
    ops.rel_pos_attention(*t)


def linear(ops, t):
    ops.linear_act_residual(t[0], t[1], t[2], residual=t[3])


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call,shapes", [
    (bias, [(32, 3)]),
    (bias_grad, [(2, 3, 4, 5)]),
    (attention, [(2, 5, 3, 64), (2, 6, 3, 64), (2, 6, 3, 64), (32, 3)]),
    (linear, [(16, 64), (32, 64), (32,), (16, 32)]),
])
def test_a_tangent_is_refused(pkg, call, shapes, grad):
    with FakeTensorMode(), fwd.dual_level():
        for n in range(len(shapes)):
            ts = [torch.zeros(*s, dtype=BF, device="cuda") for s in shapes]
            ts[n] = fwd.make_dual(ts[n].requires_grad_(grad), torch.zeros_like(ts[n]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(pkg.ops, ts)


def test_a_level_without_tangents_is_no_reason(pkg):
    with fwd.dual_level(), pytest.raises(RuntimeError, match="CUDA tensors only"):
        pkg.ops.rel_pos_bias(torch.zeros(32, 3), 4, 5)
