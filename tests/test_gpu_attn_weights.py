"""paged_attention where most of the keys carry small weights, in f16: many keys
far below a row's maximum add up to a part of the row that must not be lost.

Counted: a weight is held relative to a reference that the row's maximum is not
below, with the reference's weight at 2^7 or more, so that half of f16's
subnormal step, 2^-25, is 2^-32 of the sum that the row is divided by (that sum
is at least the maximum's weight). n keys of value v far below one key of value
zero: out = v n w / (1 + n w), off by
  u |out| for its rounding, u |out| for the weights', 4 ds |out| for the scores'
  (ds as in kv_ref), 2 n 2^-24 |out| for the sums', 2^-32 n |v| for the subnormal
  weights', and 2^-25 for a subnormal result."""
from __future__ import annotations

import math

import pytest
import torch

import higgs_amd as H

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("n", [3000, 40000, 131071, 1000000])
@pytest.mark.parametrize("below", [16.0, 17.5, 19.0])
@pytest.mark.parametrize("rows", [None, 1, 3])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_many_keys_far_below_the_maximum(dev, n, below, rows, dtype):
    """One key `below` nats above n others; rows: as a decode step, or as a
    prompt of that many tokens whose last sees n + 1 keys. The key is the first
    (a sink that draws the weight), in the middle, or the last that all rows see."""
    d, heads, page, v = 64, 2, 64, 4.0
    q = torch.zeros((rows or 1, heads, d), dtype=dtype, device=dev)
    q[..., 0] = 8.0  # scale 1/8: the score is the key's first value
    starts = None if rows is None else torch.tensor([0, rows], dtype=torch.int32, device=dev)
    n_pages = n // page + 1
    table = torch.arange(n_pages, dtype=torch.int32, device=dev)[None].contiguous()
    lens = torch.tensor([n + 1], dtype=torch.int32, device=dev)
    u = torch.finfo(dtype).eps / 2
    for at in (0, n // 2, n - 2):
        k = torch.zeros((n_pages, page, 1, d), dtype=dtype, device=dev)
        val = torch.full_like(k, v)
        k[at // page, at % page, 0, 0] = below
        val[at // page, at % page] = 0
        got = H.paged_attention(q, k, val, table, lens, q_starts=starts).double().cpu()
        for i in range(rows or 1):
            keys = n - (rows or 1) + 1 + i  # beside the one
            w = keys * math.exp(-below)
            out = v * w / (1 + w)
            ds = (d + 4) * 2.0 ** -24 * below + 2.0 ** -21 * (below + 1)
            bound = out * (2 * u + 4 * ds + 2 * keys * 2.0 ** -24)
            if dtype == F16:
                bound += 2.0 ** -32 * keys * v + 2.0 ** -25
            err = (got[i] - out).abs().max().item()
            assert err <= bound, (at, i, got[i, 0, 0].item(), out, bound)
