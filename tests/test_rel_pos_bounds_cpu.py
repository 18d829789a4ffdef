"""Arguments of the bucket rule that are no whole numbers."""
import pytest
import torch


def test_a_fractional_argument_is_refused_and_leaves_nothing_behind(pkg):
    """The rule is kept for repeated calls, where 100.0 and 100 are the same key: a refused call must
    not change what the next one gets."""
    ops = pkg.ops
    for args in ((30, 100.0, True), (30.0, 100, True), (30, 100.5, True)):
        with pytest.raises(TypeError):
            ops.rel_pos_bounds(*args)
    bounds = ops.rel_pos_bounds(30, 100, True)
    assert len(bounds) == 14 and all(type(b) is int for b in bounds)
    with pytest.raises(TypeError):
        ops.rel_pos_bias(torch.zeros(30, 2), 4, 4, max_distance=101.0)
    assert all(type(b) is int for b in ops.rel_pos_bounds(30, 101, True))
    assert ops.rel_pos_bounds(30, 100, 1) == bounds
