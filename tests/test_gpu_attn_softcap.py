"""paged_attention under soft caps from far below the scores to far above them,
against the definition in 64 bits. The bound is kv_ref's: 2^-21 (|s| + 1) for
the cap of a score s, however large the cap is, since a capped score is then
the score itself but for its own rounding."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
import kv_ref as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def run(dev, x, **kw):
    R.check(R.call(H, R.to(x, dev), **kw).cpu(), R.reference(x, **kw), str(kw))


@pytest.mark.parametrize("softcap", [64.0, 65.0, 200.0, 1e3, 1e4, 1e5, 1e6, 1e7, 1e8, 1e20, 3e38])
@pytest.mark.parametrize("news", [None, [2, 70]])
@pytest.mark.parametrize("heads,kv_heads,head_dim,dtype", [(8, 2, 64, F16), (4, 1, 96, BF16), (16, 8, 128, BF16),
                                                           (4, 2, 256, F16)])
def test_large_caps(dev, heads, kv_heads, head_dim, dtype, news, softcap):
    x = R.make(1, [300, 1030], news=news, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=16,
               dtype=dtype, q_scale=3.0)
    run(dev, x, softcap=softcap)


@pytest.mark.parametrize("softcap", [1e3, 1e5, 1e7])
@pytest.mark.parametrize("news", [None, [3]])
def test_large_caps_over_a_split_cache(dev, news, softcap):
    x = R.make(2, [9000], news=news, heads=4, kv_heads=2, head_dim=128, page=64, dtype=F16, q_scale=2.0)
    run(dev, x, softcap=softcap)
    run(dev, x, softcap=softcap, window=5000, sinks=3)


@pytest.mark.parametrize("softcap", [70.0, 300.0, 1e3])
@pytest.mark.parametrize("news", [None, [90]])
def test_large_caps_that_the_scores_reach(dev, news, softcap):
    """Scores of a few times the cap beside small ones."""
    x = R.make(3, [400], news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    for scale in (softcap * 0.03, softcap * 0.3, -softcap):
        run(dev, x, softcap=softcap, scale=scale)


@pytest.mark.parametrize("softcap", [1.0, 1e-3, 1e-20, 1e-38, 1e-40, 1e-45])
@pytest.mark.parametrize("news", [None, [40]])
def test_small_caps(dev, news, softcap):
    """Every weight is the same, also where scale / softcap is beyond f32 and a score is zero."""
    x = R.make(4, [150], news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    x["q"][:, 1] = 0
    run(dev, x, softcap=softcap)


@pytest.mark.parametrize("news", [None, [40, 150]])
def test_great_scores_under_a_greater_cap(dev, news):
    """Scores near 10^11: a cap of 10^20 changes none, one of 10^8 takes them all to its ends."""
    x = R.make(5, [333, 150], news=news, heads=4, kv_heads=2, head_dim=128, page=16, dtype=BF16, q_scale=3e5)
    x["k_pages"] *= 1e5
    d = R.to(x, dev)
    plain = R.call(H, d)
    assert torch.isfinite(plain).all()
    for cap in (1e20, 3e38):
        got = R.call(H, d, softcap=cap)
        same = (got == plain).all(-1)  # (two scores next to each other may change places in f32)
        assert torch.isfinite(got).all() and same.float().mean() > 0.98
    run(dev, x, softcap=1e8)
