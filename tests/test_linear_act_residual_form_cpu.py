"""The tile form that a product takes, for the sizes that the rule's comment in csrc/linear.cu names
(148 SMs, as without a device)."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the form of 148 SMs")


@pytest.mark.parametrize("M,N,K,b_mn,form", [
    (1024, 1536, 4096, 0, (1, 128, 1)),
    (256, 1536, 8960, 0, (1, 128, 4)),
    (2048, 1536, 8960, 0, (1, 192, 1)),
    (1024, 8960, 1536, 0, (1, 256, 1)),
    (1, 1536, 8960, 0, (0, 128, 8)),
    (1, 4096, 10240, 0, (0, 128, 4)),
    (4095, 1536, 8960, 1, (1, 192, 1)),
    (4096, 5120, 13824, 1, (1, 256, 1)),
])
def test_form_is_what_the_comment_says(pkg, M, N, K, b_mn, form):
    got = (ctypes.c_int * 3)()
    assert pkg._lib.load().wdit_linear_act_residual_form(M, N, K, b_mn, got) == 0
    assert tuple(got) == form


def test_form_refuses(pkg):
    f, got = pkg._lib.load().wdit_linear_act_residual_form, (ctypes.c_int * 3)()
    assert f(64, 64, 64, 0, None) == 1
    for M, N, K in [(0, 64, 64), (64, 0, 64), (64, 64, 0), (64, 60, 64), ((1 << 30) + 1, 64, 64), (64, 64, (1 << 30) + 8)]:
        assert f(M, N, K, 0, got) == 2


@pytest.mark.parametrize("b_mn", [0, 1])
def test_forms_fit_the_card(pkg, b_mn):
    """A split tile's CTAs run at once (74 clusters of two, 33 of four, 15 of eight), none without K blocks."""
    f, got = pkg._lib.load().wdit_linear_act_residual_form, (ctypes.c_int * 3)()
    for M in (1, 2, 17, 128, 129, 255, 300, 512, 1000, 2049, 8192, 1 << 20):
        for N in (8, 72, 264, 1536, 4104, 10240):
            for K in (8, 64, 72, 520, 4096, 13824):
                assert f(M, N, K, b_mn, got) == 0
                pair, bn, splits = got
                assert pair in (0, 1) and bn in (64, 128, 192, 256) and splits in (1, 2, 4, 8)
                assert splits <= -(-K // 64) and not (pair and (M <= 128 or bn == 64))
                group, rows = (1 + pair) * splits, -(-M // 128)
                assert group <= 8
                if splits > 1:
                    tiles = (-(-rows // 2) if pair else rows) * -(-N // bn)
                    assert tiles <= {2: 74, 4: 33, 8: 15}[group]
