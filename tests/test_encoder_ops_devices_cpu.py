"""Tensors of the text-encoder operators that lie on several devices are refused, whichever of them comes
first (fake tensors: CUDA ones without a device)."""
import itertools

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF = torch.bfloat16


def attention(ops, d, grad):
    q, k, v = (torch.empty(2, 5, 3, 64, dtype=BF, device=d[n]) for n in range(3))
    table = torch.empty(32, 3, device=d[3], requires_grad=grad)
    ops.rel_pos_attention(q, k, v, table, k_lens=torch.empty(2, dtype=torch.int32, device=d[4]))


def linear(ops, d, grad):
    x, w, r = (torch.empty(*s, dtype=BF, device=d[n]) for n, s in enumerate(((16, 64), (32, 64), (16, 32))))
    bias = torch.empty(32, device=d[3], requires_grad=grad)
    kw = {} if grad else {"out": torch.empty(16, 32, dtype=BF, device=d[4])}
    ops.linear_act_residual(x, w, bias, residual=r, **kw)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call,tensors", [(attention, 5), (linear, 5)])
@pytest.mark.parametrize("other", ["cpu", "meta"])
def test_one_tensor_elsewhere(pkg, call, tensors, other, grad):
    if call is linear and grad:
        tensors = 4
    with FakeTensorMode():
        for elsewhere in itertools.product([False, True], repeat=tensors):
            if any(elsewhere):
                devices = [other if e else "cuda" for e in elsewhere] + ["cuda"]
                with pytest.raises(RuntimeError, match="CUDA tensors only"):
                    call(pkg.ops, devices, grad)


@pytest.mark.parametrize("call", [attention, linear])
def test_two_cuda_devices(pkg, call):
    with FakeTensorMode():
        for n in range(5):
            devices = ["cuda:0"] * 5
            devices[n] = "cuda:1"
            with pytest.raises(ValueError, match="different devices"):
                call(pkg.ops, devices, False)
