"""The gradient of the table's gradient: rel_pos_bias_grad is linear in dbias, and its transpose is
rel_pos_bias."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _check_device_errors(pkg):
    yield
    pkg._lib.raise_on_device_error()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(3, 40, 50), (1, 3, 1, 1), (2, 3, 33, 64), (4, 2, 65, 7)])
def test_a_cell_gets_its_buckets_gradient(pkg, shape, dtype):
    g = torch.Generator().manual_seed(1)
    dbias = torch.randn(*shape, generator=g).to(dtype).to(DEV).requires_grad_()
    kw = dict(bidirectional=False, max_distance=30, q_offset=2)
    dtable = pkg.ops.rel_pos_bias_grad(dbias, 16, **kw)
    assert torch.equal(dtable.detach(), pkg.ops.rel_pos_bias_grad(dbias.detach(), 16, **kw))
    weight = torch.randn(dtable.shape, generator=g).to(DEV)
    (got,) = torch.autograd.grad(dtable, dbias, weight)
    want = pkg.ops.rel_pos_bias(weight.to(dtype), *shape[-2:], **kw).expand(shape)
    assert got.dtype == dtype and torch.equal(got, want)
    # the one difference there is: the op is linear
    cell = torch.zeros(shape, dtype=dtype, device=DEV)
    cell.view(-1)[-1] = 1.0
    moved = (pkg.ops.rel_pos_bias_grad(cell, 16, **kw).double() * weight.double()).sum()
    assert abs(moved.item() - got.reshape(-1)[-1].item()) <= torch.finfo(dtype).eps / 2 * abs(moved.item())


def test_it_is_not_lost_in_a_longer_run(pkg):
    """The table's gradient as a loss term: what reaches the scores' gradient, and no cells at all."""
    dbias = torch.randn(2, 3, 20, 20, device=DEV, requires_grad=True)
    (pkg.ops.rel_pos_bias_grad(dbias, 32) ** 2).sum().backward()
    with torch.no_grad():
        want = pkg.ops.rel_pos_bias(2 * pkg.ops.rel_pos_bias_grad(dbias, 32), 20, 20)
    assert torch.equal(dbias.grad, want.expand(2, 3, 20, 20))
    none = torch.randn(2, 3, 0, 20, device=DEV, requires_grad=True)
    pkg.ops.rel_pos_bias_grad(none, 32).sum().backward()
    assert none.grad.shape == none.shape
