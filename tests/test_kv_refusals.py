"""Refusals of the paged cache's calls, on the CPU: every call gives the status
of its reason."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
from higgs_amd._lib import HgkError


@pytest.mark.parametrize("dtype,head_dim", [(torch.float32, 64), (torch.bfloat16, 80), (torch.float16, 512)])
def test_what_is_not_supported_says_so(dtype, head_dim):
    """Types and head sizes that no kernel is for: status 2."""
    p = torch.zeros((4, 16, 2, head_dim), dtype=dtype)
    q = torch.zeros((2, 4, head_dim), dtype=dtype)
    t, n = torch.zeros((2, 3), dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(HgkError) as e:
        H.paged_attention(q, p, p, t, n)
    assert e.value.status == 2
    # sizes that are wrong and not unsupported keep status 1
    q = torch.zeros((2, 3, 64), dtype=torch.bfloat16)
    p = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(HgkError, match="heads") as e:
        H.paged_attention(q, p, p, t, n)
    assert e.value.status == 1


def test_a_sequence_ends_where_a_table_does():
    """2^30 tokens are the most that a call's table holds: no pages are given out beyond."""
    c = H.PagedKVCache(1, 2 ** 14 + 1, 65536, 1, 64, device="meta")
    a = c.new()
    c.extend([a], [2 ** 30 - 5])
    for n in (6, 2 ** 31):
        with pytest.raises(HgkError, match="2\\^30"):
            c.extend([a], [n])
    assert c.length(a) == 2 ** 30 - 5 and c.free_pages == 1
    c.extend([a], [5])
    assert c.length(a) == 2 ** 30
