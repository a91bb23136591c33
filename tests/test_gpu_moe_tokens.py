"""moe_route over more tokens than a launch's 2^32 threads reach."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("experts,extra", [(2, 5), (3, 16)])
def test_tokens_past_one_launch(dev, experts, extra):
    """16 tokens a block: 2^24 blocks and one or two more. The rows are windows of one run of values."""
    T = (1 << 28) + extra
    g = torch.Generator(device=dev)
    g.manual_seed(31)
    run = torch.empty(T + experts - 1, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    x = run.as_strided((T, experts), (1, 1))
    w, e = H.moe_route(x, 1)
    step = 1 << 26
    for a in range(0, T, step):
        b = min(a + step, T)
        rows = x[a:b].float()
        top, at = rows.max(1)
        same = (rows == top[:, None]).int().argmax(1).int()  # the first of equal ones
        assert torch.equal(e[a:b, 0], same), a
        p = 1.0 / torch.exp(rows - top[:, None]).sum(1)
        assert float((w[a:b, 0] - p).abs().max()) < 1e-6, a
