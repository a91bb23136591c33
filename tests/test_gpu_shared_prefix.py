"""shared_prefix_attention against paged_attention's definition in 64 bits
(tests/kv_ref.py) over tables that hold the prefix's pages."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
import kv_ref as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
LAYOUTS = [(32, 8, 64), (32, 8, 128), (16, 8, 256), (16, 2, 256), (12, 12, 64), (4, 1, 96), (28, 4, 128),
           (40, 1, 64)]


def make(seed, prefix, lens, *, news=None, **kw):
    """(inputs of the call, inputs of paged_attention with the same result). The
    call's own tables name no page in front of the prefix's end."""
    page = kw["page"]
    x = R.make(seed, [prefix, *lens], news=None if news is None else [0, *news], **kw)
    head, whole = -(-prefix // page), prefix // page
    x["prefix_table"] = x["table"][0, :head].clone()
    table, same = x["table"][1:].clone(), x["table"][1:].clone()
    table[:, :whole] = -1
    if same.shape[1] < head:
        same = torch.nn.functional.pad(same, (0, head - same.shape[1]), value=-1)
    same[:, :whole] = x["prefix_table"][:whole]
    for b, n in enumerate(lens):
        if head > whole:
            if n > prefix:  # the page that holds tokens on both sides is its own
                for name in ("k_pages", "v_pages"):
                    x[name][same[b, whole], :prefix - whole * page] = \
                        x[name][x["prefix_table"][whole], :prefix - whole * page]
            else:
                same[b, whole] = x["prefix_table"][whole]
                table[b, whole] = -1
    x["lens"] = x["lens"][1:].clone()
    if news is None:
        x["q"] = x["q"][1:].contiguous()
    else:
        x["starts"] = x["starts"][1:].clone()
    y = dict(x)
    x["table"], y["table"] = table.contiguous(), same.contiguous()
    del y["prefix_table"]
    return x, y


def call(x, prefix, **kw):
    return H.shared_prefix_attention(x["q"], x["k_pages"], x["v_pages"], x["table"], x["lens"], x["prefix_table"],
                                     prefix, q_starts=x["starts"], **kw)


def run(dev, xy, prefix, what="", **kw):
    x, y = xy
    got = call(R.to(x, dev), prefix, **kw).cpu()
    R.check(got, R.reference(y, **kw), what)
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,head_dim", LAYOUTS)
@pytest.mark.parametrize("prompts", [False, True])
def test_layouts(dev, heads, kv_heads, head_dim, dtype, prompts):
    prefix = 1000
    news = [1, 5, 33, 2, 70, 9] if prompts else None
    own = [1, 7, 40, 130, 300, 64]
    lens = [prefix + n + (news[i] if prompts else 0) for i, n in enumerate(own)]
    xy = make(1, prefix, lens, news=news, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=16, dtype=dtype)
    run(dev, xy, prefix)


@pytest.mark.parametrize("page", [1, 8, 16, 64, 256, 4096])
@pytest.mark.parametrize("prefix", [1, 63, 64, 255, 512, 1031])
@pytest.mark.parametrize("prompts", [False, True])
def test_page_sizes(dev, page, prefix, prompts):
    """Prefixes that end inside pages and inside tiles of keys."""
    lens = [prefix + 1, prefix + 3, prefix + 200]
    xy = make(2, prefix, lens, news=[1, 3, 20] if prompts else None, heads=8, kv_heads=2, head_dim=64, page=page,
              dtype=BF16)
    run(dev, xy, prefix)


@pytest.mark.parametrize("prompts", [False, True])
@pytest.mark.parametrize("prefix", [40, 700, 5000])
def test_sequences_shorter_than_the_prefix(dev, prefix, prompts):
    lens = [prefix + 9, 0, 1, prefix, prefix - 1, 17, prefix // 2 + 3, prefix + 1]
    news = [4, 0, 1, 2, 3, 17, 1, 1] if prompts else None
    xy = make(3, prefix, lens, news=news, heads=8, kv_heads=4, head_dim=128, page=16, dtype=BF16)
    got = run(dev, xy, prefix)
    if not prompts:
        assert bool((got[1] == 0).all())


@pytest.mark.parametrize("prompts", [False, True])
@pytest.mark.parametrize("softcap", [0.0, 50.0, 1.5, 200.0])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (100, 0), (100, 4), (700, 1000), (1200, 64), (2 ** 40, 0),
                                          (64, 2000), (0, 5)])
def test_windows(dev, window, sinks, softcap, prompts):
    """Windows that end in the prefix or behind it; sinks past the prefix's end."""
    prefix = 900
    news = [1, 6, 50, 130] if prompts else None
    lens = [prefix + 1, prefix + 30, prefix + 99, prefix + 500]
    xy = make(4, prefix, lens, news=news, heads=16, kv_heads=8, head_dim=128, page=16, dtype=BF16, q_scale=2.0)
    run(dev, xy, prefix, window=window, sinks=sinks, softcap=softcap)


@pytest.mark.parametrize("heads,kv_heads,head_dim,dtype", [(16, 2, 256, BF16), (32, 8, 64, F16)])
@pytest.mark.parametrize("prefix,batch,longest", [(9000, 3, 12000), (300, 70, 900), (4000, 40, 40)])
def test_long_and_wide(dev, heads, kv_heads, head_dim, dtype, prefix, batch, longest):
    """Sequences' own parts that are split and joined too, and many rows."""
    lens = [prefix + max(1, longest - 301 * i) for i in range(batch)]
    xy = make(5, prefix, lens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=32, dtype=dtype)
    run(dev, xy, prefix)


def test_one_sequence_and_no_prefix(dev):
    xy = make(6, 700, [900], heads=8, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    run(dev, xy, 700)
    xy = make(7, 0, [30, 500], heads=8, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    run(dev, xy, 0)
    x = R.to(xy[0], dev)
    x["q"], x["table"], x["lens"] = x["q"][:0], x["table"][:0], x["lens"][:0]
    assert call(x, 0).shape == (0, 8, 64)


@pytest.mark.parametrize("prompts", [False, True])
def test_sharp_scores(dev, prompts):
    """Maxima in the prefix and behind it, negative and zero scales, scores past 10^5."""
    prefix = 1500
    xy = make(8, prefix, [prefix + 400, prefix + 11], news=[7, 11] if prompts else None, heads=8, kv_heads=2,
              head_dim=128, page=64, dtype=F16, q_scale=8.0)
    for scale in (None, -0.3, 0.0):
        run(dev, xy, prefix, scale=scale)


@pytest.mark.parametrize("prompts", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values_that_are_not_finite(dev, dtype, prompts):
    """In the prefix and behind it, seen and hidden: as paged_attention."""
    prefix = 320
    news = [2, 40] if prompts else None
    lens = [prefix + 30, prefix + 90]
    x, y = make(9, prefix, lens, news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=dtype)
    v = x["v_pages"]
    v[x["prefix_table"][3], 5, 0, 7] = float("inf")
    v[x["prefix_table"][9], 1, 1, 9] = float("nan")
    v[y["table"][1, 22], 3, 0, 11] = float("-inf")
    run(dev, (x, y), prefix)
    # a window that leaves most of them out
    run(dev, (x, y), prefix, window=64, sinks=16)


def test_rows_of_no_sequence_stay(dev):
    prefix = 200
    x, y = make(10, prefix, [prefix + 3, prefix + 40], news=[3, 5], heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    x = R.to(x, dev)
    pad = torch.zeros((12, 4, 64), dtype=BF16, device=dev)
    pad[2:10] = x["q"]
    x["q"], x["starts"] = pad, x["starts"] + 2
    out = torch.full_like(pad, 7.0)
    assert call(x, prefix, out=out) is out
    assert bool((out[:2] == 7.0).all()) and bool((out[10:] == 7.0).all())
    R.check(out[2:10].cpu(), R.reference(y))


def test_strided_operands(dev):
    prefix = 130
    x, y = make(11, prefix, [prefix + 1, prefix + 70, prefix + 5], heads=8, kv_heads=2, head_dim=64, page=16, dtype=BF16,
                head_major=True)
    x = R.to(x, dev)
    wide = torch.zeros((3, 8, 192), dtype=BF16, device=dev)
    wide[:, :, 64:128] = x["q"]
    x["q"] = wide[:, :, 64:128]
    x["table"] = torch.nn.functional.pad(x["table"], (0, 5), value=3)[:, :x["table"].shape[1]]
    out = torch.zeros((8, 3, 64), dtype=BF16, device=dev).transpose(0, 1)
    call(x, prefix, out=out)
    R.check(out.cpu(), R.reference(y))


def test_pages_outside_the_pool(dev):
    """Tokens on such pages of the prefix are seen by no query."""
    prefix = 160
    x, y = make(12, prefix, [prefix + 3, prefix + 40], heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    for t in (x["prefix_table"], ):
        t[2], t[7] = -1, 10 ** 6
    y["table"][:, 2] = -1
    y["table"][:, 7] = 10 ** 6
    run(dev, (x, y), prefix)


def test_graph_replays_and_other_streams(dev):
    """Captured once, replayed over changed lengths and contents; on a stream of its own."""
    prefix = 600
    x, y = make(13, prefix, [prefix + 40, prefix + 90, prefix + 7], heads=8, kv_heads=2, head_dim=128, page=16, dtype=BF16)
    d = R.to(x, dev)
    out = torch.empty_like(d["q"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(d, prefix, out=out)
    torch.cuda.current_stream().wait_stream(s)
    R.check(out.cpu(), R.reference(y))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(d, prefix, out=out)
    for step in range(3):
        x["lens"] -= step
        d["lens"].copy_(x["lens"])
        x["q"] = (x["q"].float() * 0.9).to(BF16)
        d["q"].copy_(x["q"])
        y["lens"], y["q"] = x["lens"], x["q"]
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        R.check(out.cpu(), R.reference(y))
        assert torch.equal(call(d, prefix), out)


def test_same_bits_every_time(dev):
    x, _ = make(14, 2000, [2000 + 3 * i + 1 for i in range(20)], heads=16, kv_heads=2, head_dim=256, page=32, dtype=BF16)
    d = R.to(x, dev)
    first = call(d, 2000)
    for _ in range(3):
        assert torch.equal(first, call(d, 2000))
