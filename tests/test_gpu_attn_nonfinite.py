"""paged_attention over values that are no numbers and that its rows see: a
weight is above zero, so one infinity in a column is that infinity, both signs
are NaN, a NaN is NaN, and the other columns are what they were. Places and
signs follow the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
import kv_ref as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def plant(x, what):
    """(sequence, position, head, column, value) of the values."""
    page = x["v_pages"].shape[1]
    for b, j, h, c, value in what:
        x["v_pages"][int(x["table"][b, j // page]), j % page, h, c] = value


def compare(dev, x, **kw):
    got = R.call(H, R.to(x, dev), **kw).cpu()
    ref = R.reference(x, **kw)
    R.check(got, ref, str(kw))  # NaN places, and the finite elements
    out, _, owned = ref
    rows = owned[:, None, None].expand_as(out)
    for sign in (INF, -INF):
        assert torch.equal((got == sign) & rows, (out == sign) & rows), sign
    assert bool(torch.isinf(out).any())


@pytest.mark.parametrize("heads,kv_heads,head_dim,dtype", [(8, 2, 64, BF16), (4, 2, 96, F16), (8, 2, 128, F16),
                                                           (40, 2, 128, BF16), (4, 2, 256, BF16)])
@pytest.mark.parametrize("news", [None, [1, 40, 150]])
@pytest.mark.parametrize("q_scale", [1.0, 8.0])
@pytest.mark.parametrize("kw", [{}, {"softcap": 50.0}, {"window": 130, "sinks": 3}])
def test_seen_values_that_are_no_numbers(dev, heads, kv_heads, head_dim, dtype, news, q_scale, kw):
    """Ordinary weights, and ones of which most are too small for the type."""
    x = R.make(1, [5, 333, 150], news=news, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=16,
               dtype=dtype, q_scale=q_scale)
    last = head_dim - 1
    plant(x, [(0, 4, 0, 0, INF), (0, 2, 1, 1, -INF),
              (1, 1, 0, 5, INF), (1, 320, 0, 5, INF), (1, 300, 0, last, -INF), (1, 2, 1, 8, -INF),
              (1, 3, 1, 9, INF), (1, 210, 1, 9, -INF), (1, 290, 1, 10, NAN), (1, 292, 0, 11, NAN),
              (1, 292, 0, 12, INF), (2, 149, 0, 16, INF), (2, 0, 0, 17, INF), (2, 64, 1, 33, -INF),
              (2, 70, 1, 33, -INF), (2, 30, 0, 47, INF), (2, 100, 0, 47, -INF)])
    compare(dev, x, **kw)


@pytest.mark.parametrize("head_dim,dtype", [(64, F16), (128, BF16), (256, F16)])
@pytest.mark.parametrize("news", [None, [3]])
def test_seen_values_that_are_no_numbers_in_a_split_cache(dev, head_dim, dtype, news):
    """Parts of the keys in many blocks, joined."""
    x = R.make(2, [9000], news=news, heads=4, kv_heads=2, head_dim=head_dim, page=64, dtype=dtype, q_scale=3.0)
    plant(x, [(0, 7, 0, 0, INF), (0, 8990, 0, 1, -INF), (0, 4000, 1, 2, INF), (0, 8000, 1, 2, -INF),
              (0, 4500, 1, 3, NAN), (0, 100, 1, 40, INF), (0, 6000, 1, 40, INF)])
    compare(dev, x)
    compare(dev, x, window=6000, sinks=20)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("length", [150, 5000, 20000])
@pytest.mark.parametrize("news", [None, [2]])
def test_infinite_values_of_the_smallest_weights(dev, dtype, length, news):
    """Keys 300 nats below the maximum: no f32 holds their weight, and it is still above zero."""
    x = R.make(3, [length], news=news, heads=2, kv_heads=1, head_dim=64, page=64, dtype=dtype)
    x["q"][:] = 0
    x["q"][..., 0] = 8.0
    for e in range(x["table"].shape[1]):
        x["k_pages"][int(x["table"][0, e]), :, :, 0] = 0.0
    for top in (0, length // 2, length - 3):
        y = dict(x)
        y["k_pages"], y["v_pages"] = x["k_pages"].clone(), x["v_pages"].clone()
        y["k_pages"][int(x["table"][0, top // 64]), top % 64, :, 0] = 300.0
        plant(y, [(0, 1, 0, 3, INF), (0, length - 4, 0, 4, -INF), (0, length // 3, 0, 5, INF),
                  (0, length // 4, 0, 6, INF), (0, length - 5, 0, 6, -INF)])
        compare(dev, y)


def test_values_in_pages_that_no_row_sees_stay_out(dev):
    """Beside a row that has an infinity of its own: pages' ends, other sequences, keys in front of the window."""
    x = R.make(4, [70, 90], heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    plant(x, [(0, 3, 0, 0, INF), (0, 60, 0, 1, INF), (1, 89, 1, 2, -INF)])  # the places behind the lengths are NaN
    compare(dev, x)
    compare(dev, x, window=20)


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("head_dim,dtype", [(64, BF16), (96, F16), (128, F16), (256, BF16)])
def test_a_single_token_keeps_its_bits_beside_what_it_does_not_see(dev, bad, head_dim, dtype):
    """Keys and values in front of the window, and another sequence's."""
    x = R.make(5, [333, 90, 5000], heads=8, kv_heads=2, head_dim=head_dim, page=16, dtype=dtype)
    kw = {"window": 200, "sinks": 3}
    clean = R.call(H, R.to(x, dev), **kw).cpu()
    for pool in ("k_pages", "v_pages"):
        y = dict(x)
        y[pool] = x[pool].clone()
        for b, j in ((0, 3), (0, 100), (0, 132), (1, 60), (2, 4799)):
            y[pool][int(x["table"][b, j // 16]), j % 16, :, 5] = bad
        got = R.call(H, R.to(y, dev), **kw).cpu()
        assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2]), pool
        assert not torch.isfinite(got[1]).all()
