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


# ---------------------------------------------------------------- with a pass over the prefix
# Such small batches as above read the prefix one by one. A pass of its own is made
# from 40 MB of it on that it saves: enough sequences for that.
def many(prefix, kv_heads, head_dim):
    return 2 + (10 << 20) // (prefix * kv_heads * head_dim)


def lens_of(prefix, n, prompts, longest=90):
    """(lengths, new tokens) of n sequences behind the prefix."""
    news = [1 + 5 * i % 4 for i in range(n)] if prompts else None
    own = [(37 * i) % longest for i in range(n)]
    return [prefix + own[i] + (news[i] if prompts else 1) for i in range(n)], news


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,head_dim", LAYOUTS)
@pytest.mark.parametrize("prompts", [False, True])
def test_pass_layouts(dev, heads, kv_heads, head_dim, dtype, prompts):
    prefix = 1501
    lens, news = lens_of(prefix, many(prefix, kv_heads, head_dim), prompts)
    xy = make(21, prefix, lens, news=news, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=16, dtype=dtype)
    run(dev, xy, prefix)


@pytest.mark.parametrize("page", [1, 8, 64, 4096])
@pytest.mark.parametrize("prefix", [1023, 1024, 1087])
@pytest.mark.parametrize("prompts", [False, True])
def test_pass_page_sizes(dev, page, prefix, prompts):
    lens, news = lens_of(prefix, many(prefix, 4, 128), prompts)
    xy = make(22, prefix, lens, news=news, heads=8, kv_heads=4, head_dim=128, page=page, dtype=BF16)
    run(dev, xy, prefix)


@pytest.mark.parametrize("prompts", [False, True])
@pytest.mark.parametrize("head_dim", [64, 256])
def test_pass_over_shorter_sequences(dev, head_dim, prompts):
    prefix, n = 2100, many(2100, 4, head_dim)
    lens, news = lens_of(prefix, n, prompts)
    for i, m in enumerate((0, 1, prefix, prefix - 1, 17, prefix // 2)):
        lens[3 * i % n] = m
    if prompts:
        news = [min(a, b) for a, b in zip(news, lens)]
        news[5] = 0
    xy = make(23, prefix, lens, news=news, heads=8, kv_heads=4, head_dim=head_dim, page=16, dtype=BF16)
    got = run(dev, xy, prefix)
    if not prompts:
        assert all(bool((got[b] == 0).all()) for b, m in enumerate(lens) if m == 0)


@pytest.mark.parametrize("prompts", [False, True])
@pytest.mark.parametrize("softcap", [0.0, 50.0, 200.0])
@pytest.mark.parametrize("window,sinks", [(1, 0), (900, 64), (1300, 4), (1600, 1500), (3000, 0), (2 ** 40, 0)])
@pytest.mark.parametrize("head_dim", [128, 256])
def test_pass_windows(dev, head_dim, window, sinks, softcap, prompts):
    """Windows that end in the prefix or behind it; sinks past the prefix's end. (Those
    that hide most of the prefix take no pass.)"""
    prefix = 1400
    lens, news = lens_of(prefix, 2 * many(prefix, 8, head_dim), prompts, 400)
    xy = make(24, prefix, lens, news=news, heads=16, kv_heads=8, head_dim=head_dim, page=16, dtype=BF16, q_scale=2.0)
    run(dev, xy, prefix, window=window, sinks=sinks, softcap=softcap)


@pytest.mark.parametrize("prompts", [False, True])
@pytest.mark.parametrize("scale", [None, -0.3, 0.0, 300.0])
def test_pass_sharp_scores(dev, scale, prompts):
    """Maxima in the prefix and behind it; scores whose exponents pass 2^16."""
    prefix = 1500
    lens, news = lens_of(prefix, many(prefix, 2, 128), prompts)
    xy = make(25, prefix, lens, news=news, heads=8, kv_heads=2, head_dim=128, page=64, dtype=F16, q_scale=8.0)
    run(dev, xy, prefix, scale=scale)


@pytest.mark.parametrize("prompts", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_pass_values_that_are_not_finite(dev, head_dim, dtype, prompts):
    prefix, n = 1320, many(1320, 4, head_dim)
    lens, news = lens_of(prefix, n, prompts)
    x, y = make(26, prefix, lens, news=news, heads=8, kv_heads=4, head_dim=head_dim, page=16, dtype=dtype)
    v = x["v_pages"]
    v[x["prefix_table"][3], 5, 0, 7] = float("inf")
    v[x["prefix_table"][9], 1, 1, 9] = float("nan")
    v[x["prefix_table"][82], 7, 2, 3] = float("-inf")  # the prefix's last token
    v[y["table"][:, 82].long(), 7, 2, 3] = float("-inf")  # ... and its copies in the sequences' own pages
    v[y["table"][1, 83], 0, 0, 11] = float("-inf")     # one sequence's own
    run(dev, (x, y), prefix)
    run(dev, (x, y), prefix, window=1300, sinks=16)


def test_pass_places_and_layouts(dev):
    """Rows of no sequence, strided operands, a window's dead pages and pages outside the pool."""
    prefix = 1440
    lens, news = lens_of(prefix, many(prefix, 2, 64), True)
    x, y = make(27, prefix, lens, news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16, head_major=True)
    x["prefix_table"][2], x["prefix_table"][70] = -1, 10 ** 6
    y["table"][:, 2], y["table"][:, 70] = -1, 10 ** 6
    rows = x["q"].shape[0]
    d = R.to(x, dev)
    pad = torch.zeros((rows + 7, 4, 128), dtype=BF16, device=dev)[:, :, 64:]
    pad[3:3 + rows] = d["q"]
    d["q"], d["starts"] = pad, d["starts"] + 3
    out = torch.full((4, rows + 7, 64), 7.0, dtype=BF16, device=dev).transpose(0, 1)
    call(d, prefix, out=out)
    assert bool((out[:3] == 7).all()) and bool((out[3 + rows:] == 7).all())
    R.check(out[3:3 + rows].cpu(), R.reference(y))


@pytest.mark.parametrize("prompts", [False, True])
def test_pass_in_a_graph_and_again(dev, prompts):
    """Replays over changed lengths and queries; the same bits every time."""
    prefix = 1600
    lens, news = lens_of(prefix, many(prefix, 2, 256), prompts)
    x, y = make(28, prefix, lens, news=news, heads=16, kv_heads=2, head_dim=256, page=32, dtype=BF16)
    d = R.to(x, dev)
    out = torch.empty_like(d["q"])
    call(d, prefix, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(d, prefix, out=out)
    for step in range(3):
        x["q"] = (x["q"].float() * 0.9).to(BF16)
        d["q"].copy_(x["q"])
        if not prompts:
            x["lens"] = (x["lens"] - step).clamp(min=0)
            d["lens"].copy_(x["lens"])
        y["lens"], y["q"] = x["lens"], x["q"]
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        R.check(out.cpu(), R.reference(y))
        assert torch.equal(call(d, prefix), out)


@pytest.mark.parametrize("prompts", [False, True])
def test_pass_with_many_sequences_and_a_long_one(dev, prompts):
    """700 sequences, empty ones among them, and one whose own part is split."""
    prefix = 256
    lens, news = lens_of(prefix, 700, prompts, 30)
    lens[350] = prefix + 5000
    if not prompts:
        lens[0] = lens[699] = 0
    xy = make(29, prefix, lens, news=news, heads=4, kv_heads=2, head_dim=64, page=16, dtype=BF16)
    run(dev, xy, prefix)


@pytest.mark.parametrize("batch", [63, 65, 130, 200])
@pytest.mark.parametrize("head_dim", [64, 256])
def test_pass_with_chunks_of_ragged_sequences(dev, batch, head_dim):
    """Own parts of no chunk, of a last one only, of whole ones only and of both, in
    batches that a wave's lanes share out evenly and not."""
    prefix = 512
    own = [0, 1, 1500, 64, 0, 700, 128, 129, 33, 1024, 511, 2]
    lens = [prefix + own[(5 * i + i // 12) % 12] for i in range(batch)]
    lens[1] = lens[batch // 2] = 0
    lens[2] = 100
    xy = make(61, prefix, lens, heads=4, kv_heads=4 if head_dim == 64 else 2, head_dim=head_dim, page=16, dtype=BF16)
    run(dev, xy, prefix)
    run(dev, xy, prefix, window=900, sinks=5)


def test_pass_far_into_a_pool(dev):
    """Pages beyond 2^31 elements of the pool (and 2^32 bytes), of the prefix and of sequences."""
    prefix = 512
    lens, _ = lens_of(prefix, many(prefix, 8, 256), False)
    x, y = make(30, prefix, lens, heads=16, kv_heads=8, head_dim=256, page=64, dtype=BF16)
    n = x["k_pages"].shape[0]
    move = (1 << 31) // (64 * 8 * 256) + 11
    assert (n + move) * 64 * 8 * 256 * 2 < 6 << 30
    d = R.to({k: v for k, v in x.items() if "pages" not in k}, dev)
    for name in ("k_pages", "v_pages"):
        d[name] = torch.empty((n + move, 64, 8, 256), dtype=BF16, device=dev)
        d[name][move:] = x[name].to(dev)
    d["table"] = torch.where(d["table"] >= 0, d["table"] + move, d["table"])
    d["prefix_table"] += move
    R.check(call(d, prefix).cpu(), R.reference(y))


def test_attend_of_a_cache_with_forks(dev):
    """PagedKVCache.attend over forks, with the shared prefix it finds: as without."""
    g = torch.Generator().manual_seed(31)
    cache = H.PagedKVCache(1, 600, 16, 8, 128, device=dev)
    a = cache.new()
    cache.extend([a], [1030])
    rand = lambda n, h: torch.randn((n, h, 128), generator=g).to(BF16).to(dev)
    cache.append(0, rand(1030, 8), rand(1030, 8), cache.batch([a], [1030]))
    seqs = [a] + [cache.fork(a) for _ in range(30)]
    for step in range(3):
        cache.extend(seqs, [1] * len(seqs))
        b = cache.batch(seqs)
        cache.append(0, rand(len(seqs), 8), rand(len(seqs), 8), b)
        n = cache.shared_prefix(seqs)
        assert n == 1024
        q = rand(len(seqs), 32)
        got = cache.attend(0, q, b, prefix=n).cpu()
        k, v = cache.k_pages[0].cpu(), cache.v_pages[0].cpu()
        R.check(got, R.attend(q.cpu(), k, v, b.block_table.cpu(), b.kv_lens.cpu()))
