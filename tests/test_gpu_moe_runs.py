"""moe_route's groups where a bias holds infinities: a group whose two greatest choices
are infinities of both signs has NaN for a sum, which ranks lowest."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [4, 8])
def test_groups_whose_sum_is_not_a_number(dev, groups, scores, dtype):
    g = torch.Generator().manual_seed(41)
    x = torch.randn((5, 64), generator=g).to(dtype)
    size = 64 // groups
    bias = torch.zeros(64)
    bias[:size] = -INF
    bias[1] = INF  # group 0: inf - inf
    bias[size:2 * size] = -INF  # group 1: -inf
    w, e = H.moe_route(x.to(dev), 3, scores=scores, bias=bias.to(dev), groups=groups, top_groups=groups - 2, group_top=2)
    assert bool((e.cpu() >= 2 * size).all())
    # one more group than there are numbers: the lowest two count alike, and the lower index goes first
    w, e = H.moe_route(x.to(dev), 3, scores=scores, bias=bias.to(dev), groups=groups, top_groups=groups - 1, group_top=2)
    assert bool((e[:, 0].cpu() == 1).all()) and bool((e[:, 1:].cpu() >= 2 * size).all())
    # an infinite sum is the greatest
    bias[:size] = 0.0
    bias[1] = INF
    w, e = H.moe_route(x.to(dev), 3, scores=scores, bias=bias.to(dev), groups=groups, top_groups=1, group_top=2)
    assert bool((e.cpu() < size).all()) and bool((e[:, 0].cpu() == 1).all())
