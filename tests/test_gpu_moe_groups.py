"""The router's choice of groups where a group's two best have large biases of opposite signs: their sum is
small, and what each was rounded by is not."""
from __future__ import annotations

import pytest
import torch

import _fp8 as plain

pytestmark = pytest.mark.gpu


def same_choice(_C, x, bias, k, groups, keep, sigmoid, scale=1.0):
    w, ids = _C.moe_route(x, k, bias=bias, sigmoid=sigmoid, groups=groups, keep_groups=keep, group_best=2, scale=scale)
    ew, eids = plain.route(x, k, bias, sigmoid, groups, keep, 2, True, scale)
    assert torch.equal(ids.cpu().long(), eids)
    # one rounding to fp32, 64-bit steps before
    assert bool(((w.cpu().double() - ew).abs() <= 1.01 * 2.0 ** -24 * ew.abs()).all())


def test_two_groups_of_two(dev):
    # scores .50004 and .5 against .500025 twice: 1.00004 and 1.00005; in fp32 1000.50004 is 1000.50006 and 1000.500025 is 1000.5
    from my_int4 import _C
    s = torch.tensor([[0.50004, 0.5, 0.500025, 0.500025]], dtype=torch.float64)
    x = torch.logit(s).float().to(dev)
    for big in (1000.0, -1000.0):
        bias = torch.tensor([big, -big, big, -big], device=dev)
        w, ids = _C.moe_route(x, 2, bias=bias, sigmoid=True, groups=2, keep_groups=1, group_best=2)
        assert sorted(ids[0].tolist()) == [2, 3]
        same_choice(_C, x, bias, 2, 2, 1, True)


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("size,groups,keep", [(2, 2, 1), (2, 8, 4), (4, 16, 5), (32, 8, 3), (3, 60, 20)])
@pytest.mark.parametrize("big", [16.0, 64.0, 128.0, 1000.0, 30000.0])
def test_near_equal_groups(dev, size, groups, keep, big, sigmoid):
    from my_int4 import _C
    g = torch.Generator().manual_seed(size * groups + int(big))
    # group i has one expert of +b and one of -b, b = big (1 + i / 4), the rest are far below: single choices are far apart,
    # groups a few rounding steps of `big`
    b = big * (1 + torch.arange(groups) / 4)
    bias = torch.full((groups, size), -64 * big)
    bias[:, 0], bias[:, 1] = b, -b
    order = torch.argsort(torch.rand(groups, size, generator=g), 1)
    bias = bias.gather(1, order).reshape(-1).contiguous().to(dev)
    step = big * 2.0 ** -24 * (4.0 if sigmoid else groups * size)          # of the logits, in scores about 2^-24 big
    x = 2.0 * step * torch.randn(400, groups * size, generator=g)
    same_choice(_C, x.to(dev), bias, min(4, keep), groups, keep, sigmoid, 2.5)


def test_scores_that_64_bits_do_not_tell_apart(dev):
    """Sigmoids of 40 and 50 are both 1 in 64 bits.  Without a bias logits order experts and, by their best one, groups; sums of two
    scores and scores with a bias are equal there, and go by index."""
    from my_int4 import _C
    x = torch.tensor([[40.0, 39.0, 50.0, 45.0, 3.0, 2.0, 60.0, 1.0]], device=dev)

    def choice(k=1, **kw):
        return _C.moe_route(x, k, sigmoid=True, **kw)[1][0].tolist()

    zeros = torch.zeros(8, device=dev)
    assert choice(4) == [6, 2, 3, 0] and choice(4, bias=zeros) == [0, 1, 2, 3]
    assert choice(2, groups=4, keep_groups=2) == [6, 2] and choice(2, groups=4, keep_groups=2, bias=zeros) == [0, 1]
    assert choice(2, groups=4, keep_groups=1, group_best=2) == [0, 1] == choice(2, groups=4, keep_groups=1, group_best=2, bias=zeros)
    y = torch.tensor([[-900.0, -800.0, 0.0, -2.0, -850.0, -700.0]], device=dev)      # softmax: 0 in 64 bits below -745
    assert _C.moe_route(y, 6)[1][0].tolist() == [2, 3, 5, 1, 4, 0]
    assert _C.moe_route(y, 6, bias=torch.zeros(6, device=dev))[1][0].tolist() == [2, 3, 5, 0, 1, 4]
