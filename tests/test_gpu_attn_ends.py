"""paged_attention with sinks and a window together at the ends of int32."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
import kv_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sinks", [5, 70, 2 ** 31 - 64, 2 ** 31 - 1, 2 ** 40])
@pytest.mark.parametrize("window", [1, 20, 62, 64, 1000, 2 ** 31 - 2])
@pytest.mark.parametrize("far", [2 ** 31 - 1, 2 ** 31 - 65, 2 ** 30 + 5])
@pytest.mark.parametrize("news", [None, [1, 1], [4, 70]])
def test_sinks_of_a_length_far_beyond_the_table(dev, news, far, window, sinks):
    """The window lies behind the table (or, with the widest one, holds all of it): only sinks are seen."""
    x = R.make(1, [100, 40], news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=torch.bfloat16)
    x["k_pages"][:], x["v_pages"][:] = (torch.randn(x["k_pages"].shape).to(torch.bfloat16) for _ in range(2))
    keys = x["table"].shape[1] * 16
    x["lens"].fill_(far)
    got = R.call(H, R.to(x, dev), window=window, sinks=sinks).cpu()
    x["lens"].fill_(keys + 1200)  # as far beyond the table for these windows
    R.check(got, R.reference(x, window=window, sinks=sinks))
