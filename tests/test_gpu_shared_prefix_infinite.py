"""Infinities among the values behind a shared prefix: a row's value is the infinity
that it sees, of the right sign, however small the weight (kv_ref.check looks at NaN
and at finite results only)."""
from __future__ import annotations

import pytest
import torch

import kv_ref as R
from test_gpu_shared_prefix import BF16, F16, call, lens_of, make, many

pytestmark = pytest.mark.gpu

INF = float("inf")


def check(got, ref, what=""):
    R.check(got, ref, what)
    out, _, owned = ref
    odd = owned[:, None, None].expand_as(out) & torch.isinf(out)
    assert bool(odd.any()), f"{what}: no infinity to look at"
    g = got.to(R.F64)
    assert torch.equal(g[odd], out[odd]), f"{what}: {int((g[odd] != out[odd]).sum())} of {int(odd.sum())} infinities differ"


def put(x, y, prefix, page):
    """+inf, -inf, both and NaN in columns of their own: in the prefix, at its last token
    (and its copies in the sequences' own pages) and among one sequence's own keys."""
    v, last = x["v_pages"], (prefix - 1) // page
    places = [(x["prefix_table"][2], 5, 0, 7, INF), (x["prefix_table"][4], 0, 1, 8, -INF),
              (x["prefix_table"][0], 0, 0, 10, INF), (x["prefix_table"][5], 3, 0, 10, -INF),
              (x["prefix_table"][3], 1, 1, 9, float("nan")), (x["prefix_table"][last], (prefix - 1) % page, 1, 30, -INF),
              (y["table"][1, (prefix + 3) // page], (prefix + 3) % page, 0, 11, -INF),
              (y["table"][1, (prefix + 20) // page], (prefix + 20) % page, 1, 33, INF)]
    for page_id, at, head, col, value in places:
        v[page_id, at, head, col] = value
    own = y["table"][:, last].long()
    v[own[own >= 0], (prefix - 1) % page, 1, 30] = -INF


@pytest.mark.parametrize("prompts", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("q_scale", [1.0, 9.0])
@pytest.mark.parametrize("softcap", [0.0, 50.0])
def test_without_a_pass(dev, softcap, q_scale, dtype, prompts):
    """q_scale 9: most weights are far below what the dtype holds."""
    prefix = 325
    news = [2, 40, 1] if prompts else None
    lens = [prefix + 30, prefix + 90, prefix + 2]
    x, y = make(71, prefix, lens, news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=dtype, q_scale=q_scale)
    put(x, y, prefix, 16)
    d = R.to(x, dev)
    for kw in ({}, {"window": 64, "sinks": 48}):
        check(call(d, prefix, softcap=softcap, **kw).cpu(), R.reference(y, softcap=softcap, **kw), str(kw))


@pytest.mark.parametrize("prompts", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("head_dim,q_scale", [(64, 9.0), (96, 1.0), (128, 9.0), (256, 9.0), (128, 1.0)])
def test_with_a_pass(dev, head_dim, q_scale, dtype, prompts):
    prefix, n = 1325, many(1325, 2, head_dim)
    lens, news = lens_of(prefix, n, prompts)
    lens[1] = prefix + 60
    x, y = make(72, prefix, lens, news=news, heads=4, kv_heads=2, head_dim=head_dim, page=16, dtype=dtype, q_scale=q_scale)
    put(x, y, prefix, 16)
    d = R.to(x, dev)
    for kw in ({}, {"window": 1300, "sinks": 90}):
        check(call(d, prefix, **kw).cpu(), R.reference(y, **kw), str(kw))
