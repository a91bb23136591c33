"""The paged key-value cache on the GPU: kv_append, kv_copy_pages and
PagedKVCache, and a model-like run of them with qk_norm_rope and
paged_attention."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
import kv_ref as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def plain_append(k, pages, table, lens, starts):
    """The definition, on the CPU."""
    out = pages.clone()
    n_pages, ps = out.shape[:2]
    for b in range(lens.numel()):
        first, stop = (b, b + 1) if starts is None else (int(starts[b]), int(starts[b + 1]))
        for i in range(stop - first):
            pos = int(lens[b]) - (stop - first) + i
            if pos < 0 or pos // ps >= table.shape[1]:
                continue
            page = int(table[b, pos // ps])
            if 0 <= page < n_pages:
                out[page, pos % ps] = k[first + i]
    return out


def append_both(dev, k, v, x):
    d = R.to(x, dev)
    kd, vd = k.to(dev), v.to(dev)
    H.kv_append(kd, vd, d["k_pages"], d["v_pages"], d["table"], d["lens"], q_starts=d["starts"])
    for name, t in (("k_pages", k), ("v_pages", v)):
        want = plain_append(t, x[name], x["table"], x["lens"], x["starts"])
        got = d[name].cpu()
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)), name


@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("kv_heads,head_dim,page,dtype", [(8, 64, 16, BF16), (2, 256, 32, F16),
                                                          (1, 96, 1, BF16), (3, 128, 64, BF16)])
@pytest.mark.parametrize("news", [None, [1, 0, 37, 130]])
def test_append(dev, kv_heads, head_dim, page, dtype, news, head_major):
    lens = [1, 20, 64, 130]
    x = R.make(1, lens, news=news, heads=kv_heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
               dtype=dtype, head_major=head_major)
    k, v = (torch.randn(x["q"].shape).to(dtype) for _ in range(2))
    append_both(dev, k, v, x)


def test_append_many_rows(dev):
    """Enough rows for several units per thread."""
    x = R.make(2, [3000, 1500], news=[2999, 1000], heads=8, kv_heads=8, head_dim=128, page=64, dtype=BF16)
    k, v = (torch.randn(x["q"].shape).to(BF16) for _ in range(2))
    append_both(dev, k, v, x)


def test_append_skips_what_has_no_place(dev):
    x = R.make(3, [5, 40, 40, 33], news=[8, 3, 4, 20], heads=2, kv_heads=2, head_dim=64, page=16,
               dtype=BF16)
    n = x["k_pages"].shape[0]
    k, v = (torch.randn(x["q"].shape).to(BF16) for _ in range(2))
    x["table"][1, 2], x["table"][3, 1] = n, -1
    append_both(dev, k, v, x)  # positions below zero, pages outside the pool
    x["lens"][2] = 10 ** 9  # beyond the table
    append_both(dev, k, v, x)
    x["lens"][2] = -4
    append_both(dev, k, v, x)
    # rows in front of the first start and behind the last
    pad = [torch.randn((50, 2, 64)).to(BF16) for _ in range(2)]
    x["starts"] = x["starts"] + 4
    append_both(dev, *pad, x)
    # starts that leave the rows: those sequences are skipped, the others are not
    d = R.to(x, dev)
    before = d["k_pages"].clone()
    bad = torch.tensor([4, 12, 200, 19, 60], dtype=torch.int32, device=dev)
    H.kv_append(pad[0].to(dev), pad[1].to(dev), d["k_pages"], d["v_pages"], d["table"], d["lens"],
                q_starts=bad)
    only = dict(x, starts=torch.tensor([4, 12, 12, 12, 12], dtype=torch.int32))
    want = plain_append(pad[0], before.cpu(), x["table"], x["lens"], only["starts"])
    assert torch.equal(d["k_pages"].cpu().view(torch.int16), want.view(torch.int16))


def test_append_strided_and_layer_views(dev):
    """k and v inside a fused projection row; pages of one layer of a pool."""
    x = R.make(4, [9, 70], news=[4, 33], heads=2, kv_heads=2, head_dim=128, page=16, dtype=BF16)
    d = R.to(x, dev)
    T, n = x["q"].shape[0], x["k_pages"].shape[0]
    row = torch.randn((T, 4 + 2 + 2, 128), device=dev).to(BF16)
    pool = torch.full((3, n, 2, 16, 2, 128), 7.0, dtype=BF16, device=dev)
    kp, vp = pool[1, :, 0], pool[1, :, 1]
    H.kv_append(row[:, 4:6], row[:, 6:], kp, vp, d["table"], d["lens"], q_starts=d["starts"])
    base = torch.full((n, 16, 2, 128), 7.0, dtype=BF16)
    for got, t in ((kp, row[:, 4:6]), (vp, row[:, 6:])):
        assert torch.equal(got.cpu(), plain_append(t.cpu(), base, x["table"], x["lens"], x["starts"]))
    assert (pool[0] == 7).all() and (pool[2] == 7).all()


def test_append_offsets_past_32_bits(dev):
    step = (2 ** 32 + 4096) // 2 // 2
    pools = [torch.empty(2 * step + 16 * 64, dtype=BF16, device=dev).as_strided((3, 16, 1, 64), (step, 64, 64, 1))
             for _ in range(2)]
    for p in pools:
        p.zero_()
    table = torch.tensor([[2]], dtype=torch.int32, device=dev)
    k, v = (torch.randn((3, 1, 64), device=dev).to(BF16) for _ in range(2))
    H.kv_append(k, v, *pools, table, torch.tensor([7], dtype=torch.int32, device=dev),
                q_starts=torch.tensor([0, 3], dtype=torch.int32, device=dev))
    for p, t in zip(pools, (k, v)):
        assert torch.equal(p[2, 4:7], t) and (p[:2] == 0).all() and (p[2, :4] == 0).all()
    H.kv_copy_pages(*pools, [2], [0])
    for p in pools:
        assert torch.equal(p[0], p[2]) and (p[1] == 0).all()


# ---------------------------------------------------------------- copies
@pytest.mark.parametrize("layers", [None, 1, 3])
@pytest.mark.parametrize("order", ["tokens", "heads", "rows apart"])
@pytest.mark.parametrize("n,page,kv_heads,head_dim", [(1, 16, 8, 64), (7, 32, 2, 256), (3, 1, 1, 96),
                                                      (5, 64, 3, 128)])
def test_copy_pages(dev, layers, order, n, page, kv_heads, head_dim):
    n_pages = 2 * n + 3
    lead = () if layers is None else (layers,)
    pools = []
    for _ in range(2):
        if order == "tokens":
            t = torch.randn((*lead, n_pages, page, kv_heads, head_dim), device=dev).to(BF16)
        elif order == "heads":
            t = torch.randn((*lead, n_pages, kv_heads, page, head_dim), device=dev).to(BF16).transpose(-2, -3)
        else:
            t = torch.randn((*lead, n_pages, page, kv_heads, 2 * head_dim), device=dev).to(BF16)[..., :head_dim]
        pools.append(t)
    perm = torch.randperm(n_pages).tolist()
    src, dst = perm[:n], perm[n:2 * n]
    want = [t.clone() for t in pools]
    for w in want:
        w[..., dst, :, :, :] = w[..., src, :, :, :]
    H.kv_copy_pages(*pools, src, dst)
    for t, w in zip(pools, want):
        assert torch.equal(t, w)


def test_copy_pages_many_pairs_and_a_shared_source(dev):
    """More pairs than one launch takes; one source for several destinations."""
    n_pages = 1400
    pools = [torch.randn((n_pages, 2, 1, 64), device=dev).to(F16) for _ in range(2)]
    perm = torch.randperm(n_pages).tolist()
    src, dst = perm[:700], perm[700:]
    src[:5] = [src[0]] * 5
    want = [t.clone() for t in pools]
    for w in want:
        w[dst] = w[src]
    H.kv_copy_pages(*pools, src, dst)
    for t, w in zip(pools, want):
        assert torch.equal(t, w)
    H.kv_copy_pages(*pools, [], [])
    for t, w in zip(pools, want):
        assert torch.equal(t, w)


def test_copies_and_appends_captured(dev):
    x = R.make(5, [20, 33], heads=2, kv_heads=2, head_dim=64, page=16, dtype=BF16, spare=8)
    d = R.to(x, dev)
    k, v = (torch.randn((2, 2, 64), device=dev).to(BF16) for _ in range(2))
    free = [p for p in range(x["k_pages"].shape[0]) if p not in set(x["table"].flatten().tolist())]
    src = [int(x["table"][0, 1]), int(x["table"][1, 2])]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        H.kv_append(k, v, d["k_pages"], d["v_pages"], d["table"], d["lens"])
        H.kv_copy_pages(d["k_pages"], d["v_pages"], src, free[:2])
    for step in range(3):
        for t in (k, v):
            t.copy_(torch.randn(t.shape).to(BF16))
        d["lens"].copy_(torch.tensor([17 + step, 34 + step], dtype=torch.int32))
        want = []
        for name, t in (("k_pages", k), ("v_pages", v)):
            w = plain_append(t.cpu(), d[name].cpu(), x["table"], d["lens"].cpu(), None)
            w[free[:2]] = w[src]
            want.append(w)
        g.replay()
        torch.cuda.synchronize()
        for name, w in zip(("k_pages", "v_pages"), want):
            assert torch.equal(d[name].cpu().view(torch.int16), w.view(torch.int16)), (name, step)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("heads,kv_heads,head_dim,dims,dtype", [(8, 2, 64, 64, BF16), (4, 2, 256, 64, F16)])
def test_a_model_like_run(dev, heads, kv_heads, head_dim, dims, dtype):
    """Two layers: a prompt, forks of it that diverge token by token, a window
    layer whose dead pages are given up, compaction between steps. Every
    layer's output against the 64-bit definition over the tokens so far."""
    torch.manual_seed(7)
    layers, page, window, sinks = 2, 16, 40, 3
    cache = H.PagedKVCache(layers, 40, page, kv_heads, head_dim, dtype=dtype, device=dev)
    for t in (cache.k_pages, cache.v_pages):
        t.fill_(float("nan"))
    shadow = {}  # sequence -> per layer [keys, values] on the CPU

    def step(seqs, counts):
        cache.extend(seqs, counts)
        b = cache.batch(seqs, None if all(c == 1 for c in counts) else counts)
        T = sum(counts)
        pos = torch.cat([torch.arange(cache.length(s) - c, cache.length(s)) for s, c in zip(seqs, counts)])
        for layer in range(layers):
            q = torch.randn((T, 1, heads, head_dim), device=dev).to(dtype)
            k = torch.randn((T, 1, kv_heads, head_dim), device=dev).to(dtype)
            v = torch.randn((T, kv_heads, head_dim), device=dev).to(dtype)
            w = torch.ones(head_dim, dtype=dtype, device=dev)
            qo, ko = H.qk_norm_rope(q, k, w, w, 1e-6, dims, 1e6, offsets=pos.to(torch.int32).to(dev))
            qr, kr = qo.view(T, heads, head_dim), ko.view(T, kv_heads, head_dim)
            cache.append(layer, kr, v, b)
            kw = {"window": window, "sinks": sinks} if layer else {}
            got = cache.attend(layer, qr, b, **kw).cpu()
            at = 0
            for s, c in zip(seqs, counts):
                have = shadow.setdefault(s, [[torch.zeros((0, kv_heads, head_dim), dtype=dtype)] * 2
                                             for _ in range(layers)])
                have[layer] = [torch.cat([have[layer][0], kr[at:at + c].cpu()]),
                               torch.cat([have[layer][1], v[at:at + c].cpu()])]
                n = have[layer][0].shape[0]
                assert n == cache.length(s)
                ref = R.attend(qr[at:at + c].cpu(), have[layer][0][None], have[layer][1][None],
                               torch.zeros((1, 1), dtype=torch.int32), torch.tensor([n]),
                               torch.tensor([0, c]), **kw)
                R.check(got[at:at + c], ref, f"layer {layer} sequence {s} length {n}")
                at += c

    a, b = cache.new(), cache.new()
    step([a, b], [37, 50])
    c, e = cache.fork(a), cache.fork(a)
    for f in (c, e):
        shadow[f] = [list(t) for t in shadow[a]]
    for _ in range(3):
        step([a, b, c, e], [1, 1, 1, 1])
    cache.free(b)
    assert cache.compact() > 0
    step([c, a, e], [20, 1, 2])
    cache.free(e)
    cache.compact()
    step([a, c], [1, 1])
    used = cache.n_pages - cache.free_pages
    cache.free(a)
    cache.free(c)
    assert cache.free_pages == cache.n_pages and used > 0


def test_trimmed_pages_are_not_missed(dev):
    """With a window and sinks, giving up the pages no later query sees changes no bit."""
    torch.manual_seed(8)
    cache = H.PagedKVCache(1, 20, 16, 2, 64, device=dev)
    s = cache.new()
    cache.extend([s], [200])
    b = cache.batch([s], [200])
    cache.append(0, *(torch.randn((200, 2, 64), device=dev).to(BF16) for _ in range(2)), b)
    kw = {"window": 50, "sinks": 20}
    for _ in range(20):
        cache.extend([s], [1])
        b = cache.batch([s])
        q = torch.randn((1, 4, 64), device=dev).to(BF16)
        cache.append(0, *(torch.randn((1, 2, 64), device=dev).to(BF16) for _ in range(2)), b)
        want = cache.attend(0, q, b, **kw)
        cache.trim(s, 50, 20)
        assert torch.equal(cache.attend(0, q, cache.batch([s]), **kw), want)
    assert cache.pages(s)[:2] != [-1, -1] and cache.pages(s)[2:8].count(-1) == 6
