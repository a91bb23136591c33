"""paged_attention where scores are so great that no two of a row's are within
a softmax of each other: a row is the value of its highest score."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
import kv_ref as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype,size", [(F16, 300.0), (F16, 3e3), (F16, 1.2e4), (BF16, 300.0), (BF16, 2e4), (BF16, 1e6),
                                        (BF16, 1e9), (BF16, 1e14)])
@pytest.mark.parametrize("news", [None, [1, 40, 150]])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (4, 1, 96), (8, 2, 128), (4, 2, 256)])
def test_the_highest_score_takes_the_row(dev, heads, kv_heads, head_dim, news, dtype, size):
    x = R.make(1, [9, 333, 2300], news=news, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=16, dtype=dtype,
               q_scale=size)
    x["table"] = torch.nn.functional.pad(x["table"], (0, 900), value=-1)  # single tokens: dealt out and joined
    x["k_pages"] *= size
    got = R.call(H, R.to(x, dev)).cpu().double()
    assert torch.isfinite(got).all()
    starts = list(range(4)) if news is None else x["starts"].tolist()
    group, clear = heads // kv_heads, 0
    for b in range(3):
        n, length = starts[b + 1] - starts[b], int(x["lens"][b])
        k, _ = R.gather(x["k_pages"], x["table"][b], length)
        v, _ = R.gather(x["v_pages"], x["table"][b], length)
        for i in range(n):
            p = length - n + i
            q = x["q"][starts[b] + i].double().reshape(kv_heads, group, -1)
            s = torch.einsum("hgd,nhd->hgn", q, k[:p + 1]) / head_dim ** 0.5
            # a score is an f32 sum of D products
            ds = (head_dim + 4) * 2.0 ** -24 * torch.einsum("hgd,nhd->hgn", q.abs(), k[:p + 1].abs()).amax(-1) / head_dim ** 0.5
            row = got[starts[b] + i].reshape(kv_heads, group, -1)
            if p == 0:
                gap = torch.full_like(ds, float("inf"))
            else:
                two = s.topk(2, -1).values
                gap = two[..., 0] - two[..., 1]
            for h in range(kv_heads):
                top = v[:p + 1, h].abs().amax(0)
                for g in range(group):
                    assert (row[h, g].abs() <= top * (1 + 2.0 ** -8)).all()
                    if gap[h, g] > 2 * ds[h, g] + 120:  # the next score's weight is below any f32's
                        clear += 1
                        assert torch.equal(row[h, g], v[int(s[h, g].argmax()), h]), (b, i, h, g)
    assert clear > starts[-1] * heads // 2


@pytest.mark.parametrize("dtype,size", [(BF16, 1e20), (F16, 6e4), (BF16, float("nan")), (F16, float("inf"))])
@pytest.mark.parametrize("news", [None, [1, 40, 70]])
@pytest.mark.parametrize("kw", [{}, {"softcap": 50.0}, {"softcap": 1e4}])
def test_other_rows_keep_their_bits(dev, news, dtype, size, kw):
    """One query head (in a prompt, of one token) with such scores beside ordinary ones in a wave."""
    x = R.make(2, [9, 333, 400], news=news, heads=8, kv_heads=2, head_dim=128, page=16, dtype=dtype)
    d = R.to(x, dev)
    if dtype == F16 and size == 6e4:
        d["k_pages"] *= 500.0
    plain = R.call(H, d, **kw)
    t = 1 if news is None else 20
    d["q"][t, 2] = torch.where(d["q"][t, 2] > 0, size, -size)
    got = R.call(H, d, **kw)
    keep = torch.ones(got.shape[:2], dtype=torch.bool, device=dev)
    keep[t, 2] = False
    assert torch.equal(got[keep], plain[keep])
    if size == size and size != float("inf"):
        assert torch.isfinite(got).all() and not torch.equal(got, plain)
