"""paged_attention against its definition in 64 bits (tests/kv_ref.py), at the
sizes, masks, layouts and uses where it can go wrong."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
import kv_ref as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
LAYOUTS = [(32, 8, 64), (32, 8, 128), (16, 8, 256), (16, 2, 256), (12, 12, 64), (4, 1, 96),
           (28, 4, 128), (40, 1, 64)]


def run(dev, x, what="", **kw):
    y = R.call(H, R.to(x, dev), **kw).cpu()
    R.check(y, R.reference(x, **kw), what)
    return y


# ---------------------------------------------------------------- one token
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,head_dim", LAYOUTS)
def test_decode_layouts(dev, heads, kv_heads, head_dim, dtype):
    lens = [1, 2, 15, 16, 17, 33, 64, 65, 127, 300]
    x = R.make(1, lens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=16, dtype=dtype)
    run(dev, x)


@pytest.mark.parametrize("page", [1, 2, 8, 16, 64, 256, 4096])
@pytest.mark.parametrize("length", [1, 5, 255, 256, 257, 1031])
def test_decode_page_sizes(dev, page, length):
    x = R.make(2, [length, 3], heads=8, kv_heads=2, head_dim=128, page=page, dtype=BF16)
    run(dev, x)


@pytest.mark.parametrize("batch,length", [(1, 5000), (1, 33000), (3, 12345), (70, 700)])
def test_decode_long_and_wide(dev, batch, length):
    """Few rows over a long cache (split and joined), and many rows."""
    lens = [max(1, length - 97 * i) for i in range(batch)]
    x = R.make(3, lens, heads=8, kv_heads=2, head_dim=64, page=32, dtype=BF16)
    run(dev, x)


@pytest.mark.parametrize("kw", [{}, {"softcap": 2.0}, {"window": 1500, "sinks": 3}])
@pytest.mark.parametrize("heads,kv_heads,head_dim,dtype", [(32, 8, 64, BF16), (4, 1, 96, F16), (16, 8, 128, BF16),
                                                           (40, 2, 128, F16), (16, 2, 256, BF16)])
def test_decode_short_sequences_in_a_wide_table(dev, heads, kv_heads, head_dim, dtype, kw):
    """A table with room for long sequences: runs of tiles that end inside a pair or hold several."""
    lens = [1, 300, 0, 2, 257, 1700, 31, 0, 512, 640, 17, 900]
    x = R.make(34, lens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=16, dtype=dtype)
    x["table"] = torch.nn.functional.pad(x["table"], (0, 256), value=-1)
    run(dev, x, **kw)
    many = [1 + 37 * i % 90 for i in range(150)]
    x = R.make(35, many, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=16, dtype=dtype)
    x["table"] = torch.nn.functional.pad(x["table"], (0, 256), value=-1)
    run(dev, x, **kw)


@pytest.mark.parametrize("prompts", [False, True])
def test_many_sequences(dev, prompts):
    """More sequences than a wave has lanes, several times over, empty ones among them."""
    g = torch.Generator().manual_seed(5)
    news = torch.randint(0, 4, (700,), generator=g).tolist() if prompts else None
    lens = torch.randint(0, 90, (700,), generator=g).tolist()
    lens[0] = lens[1] = lens[699] = 0
    lens[350] = 3000
    if prompts:
        lens = [n + m for n, m in zip(lens, news)]
    x = R.make(33, lens, news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    run(dev, x)


@pytest.mark.parametrize("softcap", [0.0, 50.0, 1.5])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (100, 4), (100, 90), (64, 1000),
                                          (1000, 0), (1000, 4), (2 ** 40, 0), (0, 5)])
def test_decode_windows(dev, window, sinks, softcap):
    x = R.make(4, [1, 6, 101, 104, 105, 190, 999, 1500], heads=16, kv_heads=8, head_dim=256, page=16,
               dtype=BF16, q_scale=2.0)
    run(dev, x, window=window, sinks=sinks, softcap=softcap)


def test_decode_sharp_scores(dev):
    """Scores of large spread, maxima that keep growing and shrinking along the cache."""
    x = R.make(5, [2000, 777], heads=8, kv_heads=2, head_dim=128, page=64, dtype=F16, q_scale=8.0)
    run(dev, x)
    run(dev, x, scale=-0.3)
    run(dev, x, scale=0.0)


# ---------------------------------------------------------------- prompts
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,head_dim", LAYOUTS)
def test_prompt_layouts(dev, heads, kv_heads, head_dim, dtype):
    news, prefix = [1, 2, 31, 33, 70, 0, 129], [0, 5, 0, 64, 200, 9, 1]
    lens = [n + p for n, p in zip(news, prefix)]
    x = R.make(6, lens, news=news, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=16,
               dtype=dtype)
    run(dev, x)


@pytest.mark.parametrize("page", [1, 4, 16, 32, 128, 512])
def test_prompt_page_sizes(dev, page):
    news, lens = [150, 17, 64], [150, 300, 64]
    x = R.make(7, lens, news=news, heads=4, kv_heads=2, head_dim=64, page=page, dtype=BF16)
    run(dev, x)


@pytest.mark.parametrize("softcap", [0.0, 50.0, 1.5])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 4), (100, 90), (64, 1000),
                                          (300, 0), (129, 65), (0, 5)])
def test_prompt_windows(dev, window, sinks, softcap):
    news, lens = [290, 40, 3], [290, 401, 130]
    x = R.make(8, lens, news=news, heads=4, kv_heads=2, head_dim=128, page=16, dtype=BF16, q_scale=2.0)
    run(dev, x, window=window, sinks=sinks, softcap=softcap)


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(4, 4, 64), (8, 1, 128), (2, 1, 256), (3, 1, 96)])
def test_prompt_few_rows_over_a_long_cache(dev, heads, kv_heads, head_dim):
    """A short turn over a long prefix: split over the cache and joined."""
    x = R.make(9, [9000, 4100], news=[5, 20], heads=heads, kv_heads=kv_heads, head_dim=head_dim,
               page=64, dtype=BF16)
    run(dev, x)
    run(dev, x, window=3000, sinks=3)


def test_prompt_longer(dev):
    x = R.make(10, [700, 513], news=[700, 511], heads=8, kv_heads=2, head_dim=128, page=64, dtype=F16,
               q_scale=4.0)
    run(dev, x)


def test_prompt_of_one_token_each_equals_decode(dev):
    """The two forms of a call of single tokens agree within their bounds."""
    lens = [1, 50, 333]
    x = R.make(11, lens, heads=8, kv_heads=2, head_dim=128, page=16, dtype=BF16)
    run(dev, x)
    x["starts"] = torch.arange(4, dtype=torch.int32)
    run(dev, x)


# ---------------------------------------------------------------- masks and odd data
def test_rows_that_see_nothing_are_zero(dev):
    x = R.make(12, [0, 5, 0], heads=8, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    y = run(dev, x)
    assert (y[0] == 0).all() and (y[2] == 0).all() and not (y[1] == 0).all()
    # more new tokens than the length counts: the first rows lie before the sequence
    x = R.make(13, [3, 0, 70], news=[10, 4, 200], heads=4, kv_heads=2, head_dim=128, page=16, dtype=F16)
    y = run(dev, x)
    assert (y[:7] == 0).all() and not (y[7] == 0).all() and (y[10:14] == 0).all()
    # a negative length counts as none
    x["lens"][2] = -5
    y = run(dev, x)
    assert (y[14:] == 0).all()


@pytest.mark.parametrize("news", [None, [40, 1, 130]])
def test_pages_outside_the_pool_are_not_seen(dev, news):
    lens = [40, 200, 333]
    x = R.make(14, lens, news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    n = x["k_pages"].shape[0]
    for b, e, bad in ((0, 0, -1), (1, 3, n), (1, 11, 2 ** 31 - 1), (2, 0, -2 ** 31), (2, 20, -7)):
        x["table"][b, e] = bad
    y = run(dev, x)
    if news:
        assert (y[:16] == 0).all()
    x["table"][:] = n + 5
    assert (run(dev, x) == 0).all()
    # a length beyond the table ends at the table; none at all is nothing seen
    x = R.make(15, lens, news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    x["table"] = x["table"][:, :9].contiguous()
    run(dev, x)
    x["table"] = x["table"][:, :0].contiguous()
    assert (run(dev, x) == 0).all()


def test_starts_outside_the_rows_reach_nothing(dev):
    x = R.make(16, [20, 30], news=[8, 8], heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    for starts in ([0, 8, 17], [-3, 8, 16], [0, 2 ** 31 - 1, 16], [8, 8, 8], [16, 8, 0]):
        d = R.to(x, dev)
        d["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        out = torch.full_like(d["q"], 7.0)
        R.call(H, d, out=out)
        y = out.cpu()
        for b in range(2):
            lo, hi = starts[b], starts[b + 1]
            if 0 <= lo < hi <= 16:
                assert not (y[lo:hi] == 7).all()
        covered = [t for b in range(2) if 0 <= starts[b] < starts[b + 1] <= 16
                   for t in range(starts[b], starts[b + 1])]
        rest = [t for t in range(16) if t not in covered]
        assert (y[rest] == 7).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("head_dim,dtype", [(64, BF16), (128, F16), (256, BF16)])
def test_values_that_are_not_seen_do_not_reach_a_row(dev, bad, head_dim, dtype):
    """A key or value that is no number: rows that do not see it keep their bits."""
    unseen(dev, bad, head_dim, dtype, 16, ({}, {"window": 40, "sinks": 3}))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("head_dim,dtype,page", [(64, BF16, 4), (96, F16, 2), (128, BF16, 16), (256, F16, 4)])
def test_values_that_are_not_seen_with_a_soft_cap(dev, bad, head_dim, dtype, page):
    """The same, capped, and with pages that end inside a tile's rows."""
    unseen(dev, bad, head_dim, dtype, page, ({"softcap": 50.0}, {"softcap": 2.0, "window": 40, "sinks": 3}))


def unseen(dev, bad, head_dim, dtype, page, masks):
    news, lens = [150, 90], [150, 400]
    x = R.make(17, lens, news=news, heads=4, kv_heads=2, head_dim=head_dim, page=page, dtype=dtype)
    for kw in masks:
        clean = run(dev, x, **kw)
        for pool in ("k_pages", "v_pages"):
            for b, j in ((0, 77), (0, 149), (1, 330)):
                y = dict(x)
                y[pool] = x[pool].clone()
                y[pool][int(x["table"][b, j // page]), j % page, :, 5] = bad
                got = R.call(H, R.to(y, dev), **kw).cpu()
                for s, (n, length) in enumerate(zip(news, lens)):
                    first = 0 if s == 0 else news[0]
                    for i in range(n):
                        p = length - n + i
                        sees = s == b and bool(R.seen_mask(p, length, kw.get("window", 0),
                                                           kw.get("sinks", 0))[j])
                        row, ref = got[first + i], clean[first + i]
                        if not sees:
                            assert torch.equal(row, ref), (pool, b, j, s, i)
                        elif pool == "v_pages":
                            # p > 0 of an infinite or NaN value, in that column alone
                            assert not torch.isfinite(row[:, 5]).any(), (b, j, s, i)
                            rest = [c for c in range(head_dim) if c != 5]
                            assert torch.isfinite(row[:, rest]).all(), (b, j, s, i)


def test_infinite_scores_follow_the_formula(dev):
    """All seen scores -inf, or one +inf: 0/0, NaN; seen -inf beside finite ones: weight 0."""
    x = R.make(18, [3, 40], heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    x["q"][:] = 1.0
    for b, j in ((0, 0), (0, 1), (0, 2), (1, 7)):
        x["k_pages"][int(x["table"][b, j // 16]), j % 16, :, 0] = float("-inf")
    y = R.call(H, R.to(x, dev)).cpu()
    assert torch.isnan(y[0]).all() and torch.isfinite(y[1]).all()
    x["starts"] = torch.tensor([0, 1, 2], dtype=torch.int32)
    y2 = R.call(H, R.to(x, dev)).cpu()
    assert torch.isnan(y2[0]).all() and torch.isfinite(y2[1]).all()
    R.check(y2, R.reference(x))
    x["k_pages"][int(x["table"][1, 0]), 7, :, 0] = float("inf")
    for starts in (None, x["starts"]):
        x["starts"] = starts
        assert torch.isnan(R.call(H, R.to(x, dev)).cpu()[1]).all()


@pytest.mark.parametrize("news", [None, [3]])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_many_small_weights_beside_a_large_one(dev, news, dtype):
    """One key of weight 1 and 6000 of about e^-10 each, subnormal in f16: their
    sum is a quarter of the whole and none of it may be lost. Bound as ever."""
    x = R.make(31, [6001], news=news, heads=4, kv_heads=2, head_dim=64, page=64, dtype=dtype)
    x["q"][:] = 0
    x["q"][..., 0] = 8.0
    for e in range(x["table"].shape[1]):
        x["k_pages"][int(x["table"][0, e]), :, :, 0] = 0.0
    x["k_pages"][int(x["table"][0, 1]), 5, :, 0] = 10.0  # score 80 / 8 = 10, the others 0
    run(dev, x)


@pytest.mark.parametrize("news", [None, [4, 70]])
def test_lengths_at_the_ends_of_their_type(dev, news):
    """Lengths far beyond the table (its keys, all in front of the queries, are
    seen without a window, and not with one) and below zero."""
    lens = [4, 100]
    x = R.make(32, lens, news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    x["k_pages"][:], x["v_pages"][:] = (torch.randn(x["k_pages"].shape).to(BF16) for _ in range(2))
    d = R.to(x, dev)
    for far in (2 ** 31 - 1, 2 ** 30 + 5):
        d["lens"].fill_(far)
        y = R.call(H, d).cpu()
        for window, same in ((0, True), (2 ** 31 - 1, True), (2 ** 31, True), (1000, False)):
            z = R.call(H, d, window=window).cpu()
            assert torch.equal(z, y) if same else (z == 0).all()
        k = x["table"].shape[1] * 16
        short = {**x, "lens": torch.tensor([k + 200, k + 200], dtype=torch.int32)}
        R.check(y, R.reference(short))
    d["lens"].fill_(-2 ** 31)
    assert (R.call(H, d).cpu() == 0).all()


# ---------------------------------------------------------------- layouts
@pytest.mark.parametrize("news", [None, [40, 1, 130]])
@pytest.mark.parametrize("head_major", [False, True])
def test_strided_operands(dev, news, head_major):
    lens = [40, 200, 333]
    x = R.make(19, lens, news=news, heads=8, kv_heads=2, head_dim=128, page=16, dtype=BF16,
               head_major=head_major)
    d = R.to(x, dev)
    T = d["q"].shape[0]
    # q inside a fused projection row, out head-major inside a larger buffer, table with a stride
    fused = torch.full((T, 8 + 2 + 2, 128), float("nan"), dtype=BF16, device=dev)
    fused[:, :8] = d["q"]
    d["q"] = fused[:, :8]
    buf = torch.full((8, T + 3, 128), 7.0, dtype=BF16, device=dev)
    wide = torch.full((3, d["table"].shape[1] + 5), 10 ** 6, dtype=torch.int32, device=dev)
    wide[:, :-5] = d["table"]
    d["table"] = wide[:, :-5]
    out = buf[:, :T].transpose(0, 1)
    assert R.call(H, d, out=out) is out
    R.check(out.cpu(), R.reference(x))
    assert (buf[:, T:] == 7).all()
    # keys and values of one pool [n_pages, 2, page_size, Hk, D]
    both = torch.stack([d["k_pages"], d["v_pages"]], 1)
    d["k_pages"], d["v_pages"] = both[:, 0], both[:, 1]
    R.check(R.call(H, d).cpu(), R.reference(x))
    # one kv head for all, by a stride of zero
    x1 = R.make(20, lens, news=news, heads=8, kv_heads=1, head_dim=64, page=16, dtype=BF16)
    d = R.to(x1, dev)
    d["k_pages"], d["v_pages"] = (d[n].expand(-1, -1, 4, -1) for n in ("k_pages", "v_pages"))
    R.check(R.call(H, d).cpu(), R.reference(x1))


def test_rows_of_no_sequence_are_left_alone(dev):
    """A padded batch: rows in front of the first start and behind the last."""
    x = R.make(21, [30, 64], news=[7, 40], heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    d = R.to(x, dev)
    pad = torch.randn((60, 4, 64), device=dev).to(BF16)
    pad[5:52] = d["q"]
    d["q"], d["starts"] = pad, d["starts"] + 5
    out = torch.full_like(pad, 7.0)
    R.call(H, d, out=out)
    R.check(out[5:52].cpu(), R.reference(x))
    assert (out[:5] == 7).all() and (out[52:] == 7).all()


@pytest.mark.parametrize("news", [None, [70]])
def test_offsets_past_32_bits(dev, news):
    """Pages that lie more than 2^32 bytes apart."""
    x = R.make(22, [300], news=news, heads=4, kv_heads=1, head_dim=64, page=128, dtype=BF16, spare=0)
    d = R.to(x, dev)
    step = (2 ** 32 + 4096) // 2 // 2  # elements: the third page is past 2^32 bytes
    for name in ("k_pages", "v_pages"):
        big = torch.empty(2 * step + 128 * 64, dtype=BF16, device=dev)
        view = big.as_strided((3, 128, 1, 64), (step, 64, 64, 1))
        view.copy_(d[name])
        d[name] = view
    R.check(R.call(H, d).cpu(), R.reference(x))


# ---------------------------------------------------------------- use
@pytest.mark.parametrize("news", [None, [5, 60]])
def test_calls_repeat_bit_for_bit(dev, news):
    x = R.make(23, [9000, 4000], news=news, heads=8, kv_heads=2, head_dim=64, page=64, dtype=BF16)
    d = R.to(x, dev)
    y = R.call(H, d)
    for _ in range(3):
        assert torch.equal(R.call(H, d), y)


def test_calls_on_two_streams_at_once(dev):
    x = [R.make(24 + i, [9000 - i, 4000], heads=8, kv_heads=2, head_dim=64, page=64, dtype=BF16)
         for i in range(2)]
    d = [R.to(t, dev) for t in x]
    alone = [R.call(H, t) for t in d]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(R.call(H, d[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, alone[i])


@pytest.mark.parametrize("news", [None, [5, 60]])
def test_captured_and_replayed(dev, news):
    """Two graphs of the same call, replayed over new lengths, tables and data, with eager work between."""
    x = R.make(26, [9000, 4000], news=news, heads=8, kv_heads=2, head_dim=64, page=64, dtype=BF16)
    d = R.to(x, dev)
    R.call(H, d)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(R.call(H, d, window=5000, sinks=4))
        graphs.append(g)
    for step in range(4):
        if news is None or step % 2:
            d["lens"].copy_(torch.tensor([8000 - 1111 * step, 70 + step], dtype=torch.int32))
        d["q"].copy_(torch.randn(d["q"].shape).to(BF16))
        d["table"].copy_(d["table"].roll(1, 1) if step == 2 else d["table"])
        eager = R.call(H, d, window=5000, sinks=4)
        torch.cuda.synchronize()
        for g, o in zip(graphs, outs):
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o.isnan(), eager.isnan())
            assert torch.equal(o.nan_to_num(), eager.nan_to_num()), step


def test_empty_calls(dev):
    x = R.make(27, [5], heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    d = R.to(x, dev)
    d["q"], d["table"], d["lens"] = d["q"][:0], d["table"][:0], d["lens"][:0]
    assert R.call(H, d).shape == (0, 4, 64)
    d = R.to(x, dev)
    d["starts"] = torch.zeros(2, dtype=torch.int32, device=dev)
    d["q"] = d["q"][:0]
    assert R.call(H, d).shape == (0, 4, 64)
    # no sequence, but rows: they belong to none
    d = R.to(x, dev)
    d["starts"], d["table"], d["lens"] = (torch.zeros(1, dtype=torch.int32, device=dev), d["table"][:0],
                                          d["lens"][:0])
    out = torch.full_like(d["q"], 7.0)
    R.call(H, d, out=out)
    assert (out == 7).all()
