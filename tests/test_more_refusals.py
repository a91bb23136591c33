"""Refusals of the shared prefix's attention, of pages given out on the GPU, of slot
maps and of the experts' routing and sum, on the CPU: no such call reaches a kernel."""
from __future__ import annotations

import ctypes as C
import shutil
import subprocess

import pytest
import torch

import higgs_amd as H
from higgs_amd import _lib, ops
from higgs_amd._lib import HgkError, HgkKvBatch, HgkKvPages, HgkKvTables

FAKE = 1 << 20  # never dereferenced
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def st(*v):
    return (C.c_int64 * len(v))(*v)


def pages(**kw):
    d = dict(dtype=1, page_size=16, n_pages=8, kv_heads=2, head_dim=64, k=FAKE, v=FAKE,
             k_strides=st(2048, 128, 64), v_strides=st(2048, 128, 64))
    return HgkKvPages(**{**d, **kw})


def batch(**kw):
    d = dict(batch=2, tokens=2, block_table=FAKE, table_stride=4, table_width=4, kv_lens=FAKE, q_starts=None)
    return HgkKvBatch(**{**d, **kw})


def shared(p=None, b=None, table=FAKE, width=2, prefix=20, q=FAKE, qs=(256, 64), heads=4, scale=0.125, softcap=0.0,
           window=0, sinks=0, out=FAKE, os_=(256, 64), ws=None, n=0):
    L = _lib.lib()
    s = L.hgk_shared_prefix_attention(C.byref(p or pages()), C.byref(b or batch()), table, width, prefix, q, st(*qs),
                                      heads, scale, softcap, window, sinks, out, st(*os_), ws, n, None)
    return s, L.hgk_last_error().decode()


def test_struct_layout():
    """ctypes, the packed form the Python calls use, and the C header agree."""
    assert C.sizeof(HgkKvTables) == ops._KV_TABLES.size
    got = HgkKvTables.from_buffer_copy(ops._KV_TABLES.pack(1, 2, 3, 4, 5, 6, 7, 8, 9))
    assert [getattr(got, f[0]) for f in HgkKvTables._fields_] == list(range(1, 10))
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc:
        import os
        import tempfile

        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        src = "#include <stdio.h>\n#include <stddef.h>\n#include \"higgs_hip.h\"\nint main(void){printf(\"%zu \", sizeof(hgk_kv_tables));"
        for f in HgkKvTables._fields_:
            src += f"printf(\"%zu \", offsetof(hgk_kv_tables, {f[0]}));"
        with tempfile.TemporaryDirectory() as d:
            open(os.path.join(d, "l.c"), "w").write(src + "return 0;}\n")
            subprocess.run([cc, "-I", os.path.join(root, "include"), os.path.join(d, "l.c"), "-o", os.path.join(d, "l")],
                           check=True)
            out = subprocess.run([os.path.join(d, "l")], capture_output=True, text=True, check=True).stdout
        assert [int(v) for v in out.split()] == [C.sizeof(HgkKvTables),
                                                 *(getattr(HgkKvTables, f[0]).offset for f in HgkKvTables._fields_)]


@pytest.mark.parametrize("kw,status,text", [
    (dict(p=pages(dtype=0)), 2, "bf16 or f16"), (dict(p=pages(head_dim=80)), 2, "head_dim"),
    (dict(p=pages(page_size=24)), 1, "page_size"), (dict(b=batch(tokens=3)), 1, "3 rows"),
    (dict(b=batch(kv_lens=None)), 1, "null"), (dict(heads=3), 1, "heads"), (dict(window=-1), 1, "window"),
    (dict(sinks=-1), 1, "sinks"), (dict(prefix=-1), 1, "prefix"), (dict(prefix=33), 1, "do not hold"),
    (dict(width=0), 1, "do not hold"), (dict(width=-1), 1, "prefix"), (dict(width=1 << 27), 1, "prefix"),
    (dict(prefix=(1 << 30) + 1, width=1 << 26), 1, "prefix"), (dict(table=None), 1, "null prefix table"),
    (dict(scale=float("nan")), 1, "scale"), (dict(softcap=-1.0), 1, "softcap"), (dict(q=None), 1, "null q"),
    (dict(out=None), 1, "null out"), (dict(q=FAKE + 8), 1, "aligned"), (dict(os_=(0, 64)), 1, "overlap"),
])
def test_refused_shared_prefix(kw, status, text):
    s, msg = shared(**kw)
    assert s == status and text in msg, (s, msg)


def test_shared_prefix_workspace():
    L = _lib.lib()

    def need(p=None, b=None, width=2, prefix=20, heads=4, window=0, sinks=0):
        return L.hgk_shared_prefix_attention_workspace(C.byref(p or pages()), C.byref(b or batch()), width, prefix, heads,
                                                       window, sinks)

    assert need() == 0  # a small call has no second pass
    for kw in (dict(heads=3), dict(prefix=33), dict(width=-1), dict(window=-1), dict(p=pages(head_dim=80))):
        assert need(**kw) == -1
    long = batch(batch=64, tokens=64, table_width=2048, table_stride=2048)
    kw = dict(b=long, width=1024, prefix=16384)
    n = need(**kw)
    assert n > 0
    for ws, m in ((None, n), (FAKE, n - 1), (FAKE + 4, n)):
        s, msg = shared(ws=ws, n=m, **kw)
        assert s == 1 and "workspace" in msg
    for b in (batch(batch=0, tokens=0), batch(batch=3, tokens=0, q_starts=FAKE)):
        assert need(b=b) == 0 and shared(b=b, q=None, out=None)[0] == 0


def tables(**kw):
    d = dict(page_size=16, rows=4, tables=FAKE, table_stride=8, table_width=8, lens=FAKE, free_pages=FAKE, n_pages=30,
             n_free=FAKE)
    return HgkKvTables(**{**d, **kw})


def extend(t=None, seqs=FAKE, counts=FAKE, n=2, tokens=5, lens=FAKE, free=FAKE, kv=FAKE, starts=FAKE, slots=FAKE,
           pos=FAKE, bt=FAKE, stride=8, status=FAKE, ws=FAKE):
    L = _lib.lib()
    s = L.hgk_kv_extend(C.byref(t or tables()), seqs, counts, n, tokens, lens, free, kv, starts, slots, pos, bt, stride,
                        status, ws, None)
    return s, L.hgk_last_error().decode()


def release(t=None, seqs=FAKE, keep=None, owned=None, n=2, lens=FAKE, free=FAKE, status=FAKE, ws=FAKE):
    L = _lib.lib()
    s = L.hgk_kv_release(C.byref(t or tables()), seqs, keep, owned, n, lens, free, status, ws, None)
    return s, L.hgk_last_error().decode()


@pytest.mark.parametrize("kw,status,text", [
    (dict(page_size=0), 1, "page_size"), (dict(page_size=24), 1, "page_size"), (dict(page_size=1 << 17), 1, "page_size"),
    (dict(rows=-1), 1, "rows"), (dict(rows=(1 << 18) + 1), 2, "rows"), (dict(n_pages=-1), 1, "n_pages"),
    (dict(n_pages=1 << 31), 1, "n_pages"), (dict(table_width=-1), 1, "width"), (dict(table_stride=7), 1, "stride"),
    (dict(table_stride=-8), 1, "stride"), (dict(table_width=1 << 27, table_stride=1 << 27), 1, "too wide"),
    (dict(lens=None), 1, "null"), (dict(tables=None), 1, "null"), (dict(free_pages=None), 1, "null"),
    (dict(n_free=None), 1, "null"),
])
def test_refused_tables(kw, status, text):
    for call in (extend, release):
        s, msg = call(t=tables(**kw))
        assert s == status and text in msg, (s, msg)


def test_refused_steps():
    for kw, text in ((dict(seqs=None, bt=None), "numbers"), (dict(n=5), "5 sequences"), (dict(n=-1), "batch"),
                     (dict(tokens=-1), "tokens"), (dict(tokens=(1 << 30) + 1), "tokens"), (dict(counts=None), "null"),
                     (dict(lens=None), "null"), (dict(free=None), "null"), (dict(kv=None), "null"),
                     (dict(starts=None), "null"), (dict(slots=None), "null"), (dict(pos=None), "null"),
                     (dict(status=None), "null"), (dict(ws=None), "null"), (dict(stride=7), "overlap"),
                     (dict(seqs=None, n=4), "numbers")):
        s, msg = extend(**kw)
        assert s == 1 and text in msg, (kw, msg)
    for kw, text in ((dict(seqs=None), "numbers"), (dict(n=5), "5 sequences"), (dict(lens=None), "null"),
                     (dict(free=None), "null"), (dict(status=None), "null"), (dict(ws=None), "null")):
        s, msg = release(**kw)
        assert s == 1 and text in msg, (kw, msg)
    assert _lib.lib().hgk_kv_extend(None, *[None] * 2, 0, 0, *[None] * 7, 0, None, None, None) == 1


def test_refused_slots():
    L = _lib.lib()
    ok = dict(p=pages(), slots=FAKE, n=3, ks=(128, 64))

    def call(**kw):
        d = {**ok, **kw}
        s = L.hgk_kv_append_slots(C.byref(d["p"]), d["slots"], d["n"], FAKE, st(*d["ks"]), FAKE + (1 << 30), st(128, 64), None)
        return s, L.hgk_last_error().decode()

    # (pages whose keys lie on their values are refused as in hgk_kv_append)
    assert call()[0] == 1 and "overlap" in call()[1]
    apart = pages(v=FAKE + (1 << 24))
    for kw, text in ((dict(slots=None), "slots"), (dict(slots=FAKE + 4), "slots"), (dict(n=-1), "tokens"),
                     (dict(n=1 << 31), "tokens"), (dict(ks=(128, 60)), "multiples")):
        s, msg = call(**{"p": apart, **kw})
        assert s == 1 and text in msg, (kw, msg)
    assert call(p=pages(dtype=0))[0] == 2
    assert L.hgk_kv_append_slots(C.byref(apart), None, 0, None, None, None, None, None) == 0


def test_slots_in_place_of_tables():
    p = torch.zeros((4, 16, 2, 64), dtype=BF16)
    k, v = torch.zeros((3, 2, 64), dtype=BF16), torch.zeros((3, 2, 64), dtype=BF16)
    s = torch.zeros(3, dtype=torch.int64)
    t, n = torch.zeros((3, 2), dtype=I32), torch.ones(3, dtype=I32)
    for kw in (dict(slots=s, block_table=t), dict(slots=s, kv_lens=n), dict(slots=s, q_starts=n)):
        with pytest.raises(HgkError, match="in place of"):
            H.kv_append(k, v, p, p, **kw)
    for bad in (s[:2], s.to(I32), torch.zeros(6, dtype=torch.int64)[::2]):
        with pytest.raises(HgkError, match="slots must be"):
            H.kv_append(k, v, p, p, slots=bad)
    for kw in ({}, dict(block_table=t), dict(kv_lens=n)):
        with pytest.raises(HgkError, match="must be given"):
            H.kv_append(k, v, p, p, **kw)
    with pytest.raises(HgkError, match="GPU"):
        H.kv_append(k, v, p, torch.zeros_like(p), slots=s)


def route(dtype=1, logits=FAKE, stride=64, bias=None, scores=0, tokens=4, n=64, k=8, groups=1, top_groups=1, group_top=1,
          scale=1.0, weights=FAKE, experts=FAKE):
    L = _lib.lib()
    s = L.hgk_moe_route(dtype, logits, stride, bias, scores, tokens, n, k, groups, top_groups, group_top, 0, scale, weights,
                        experts, None)
    return s, L.hgk_last_error().decode()


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=4), 1, "dtype"), (dict(dtype=9), 1, "dtype"), (dict(scores=2), 1, "scores"), (dict(tokens=-1), 1, "tokens"),
    (dict(tokens=1 << 31), 1, "too many"), (dict(n=0), 1, "experts"), (dict(n=1025), 2, "experts"), (dict(k=0), 1, "top_k"),
    (dict(k=65), 1, "top_k"), (dict(n=128, k=65), 2, "top_k"), (dict(groups=0), 1, "groups"), (dict(groups=7), 1, "groups"),
    (dict(groups=8, top_groups=0), 1, "groups"), (dict(groups=8, top_groups=9), 1, "groups"),
    (dict(n=260, groups=65, top_groups=65), 2, "groups"), (dict(groups=16, top_groups=1), 1, "top_k"),
    (dict(group_top=3), 1, "group_top"), (dict(group_top=0), 1, "group_top"),
    (dict(groups=64, top_groups=8, group_top=2), 1, "group_top"), (dict(n=1020, groups=51, top_groups=2), 2, "groups"),
    (dict(scale=float("inf")), 1, "scale"), (dict(scale=float("nan")), 1, "scale"), (dict(stride=-64), 1, "stride"),
    (dict(logits=None), 1, "null"), (dict(weights=None), 1, "null"), (dict(experts=None), 1, "null"),
    (dict(logits=FAKE + 1), 1, "aligned"), (dict(bias=FAKE + 2), 1, "aligned"), (dict(experts=FAKE + 2), 1, "aligned"),
])
def test_refused_routes(kw, status, text):
    s, msg = route(**kw)
    assert s == status and text in msg, (s, msg)


def test_empty_routes_and_sums():
    assert route(tokens=0, logits=None, weights=None, experts=None)[0] == 0
    assert combine(tokens=0, y=None, w=None, out=None)[0] == 0
    assert combine(hidden=0, y=None, w=None, out=None)[0] == 0


def combine(dtype=1, y=FAKE, ys=64, w=FAKE, wst=2, k=2, shared=None, ss=64, gate=None, gd=1, gs=1, out=FAKE, os_=64,
            tokens=4, hidden=64):
    L = _lib.lib()
    s = L.hgk_moe_combine(dtype, y, ys, w, wst, k, shared, ss, gate, gd, gs, out, os_, tokens, hidden, None)
    return s, L.hgk_last_error().decode()


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype"), (dict(tokens=-1), "tokens"), (dict(hidden=-1), "hidden"), (dict(k=0), "top_k"),
    (dict(gate=FAKE), "gate without"), (dict(shared=FAKE, gate=FAKE, gd=4), "gate of dtype"), (dict(y=None), "null"),
    (dict(w=None), "null"), (dict(out=None), "null"), (dict(y=FAKE + 1), "aligned"), (dict(w=FAKE + 2), "aligned"),
    (dict(shared=FAKE + 1), "aligned"), (dict(shared=FAKE, gate=FAKE + 1), "aligned"), (dict(ys=-64), "stride"),
    (dict(wst=-1), "stride"), (dict(os_=63), "overlap"), (dict(os_=0), "overlap"), (dict(tokens=1 << 30, k=4), "too many"),
])
def test_refused_sums(kw, text):
    s, msg = combine(**kw)
    assert s == 1 and text in msg, (s, msg)


def test_python_refusals():
    """What the Python calls check before the library is asked."""
    x = torch.zeros((4, 64), dtype=BF16)
    for kw, text in ((dict(scores="relu"), "scores"), (dict(bias=torch.zeros(63)), "bias"),
                     (dict(bias=torch.zeros(64, dtype=BF16)), "bias"), (dict(bias=torch.zeros(128)[::2]), "bias")):
        with pytest.raises(HgkError, match=text):
            H.moe_route(x, 2, **kw)
    for k in (0, -1, 65):
        with pytest.raises(HgkError, match="top_k"):
            H.moe_route(x, k)
    with pytest.raises(HgkError, match="unit-stride"):
        H.moe_route(x.t(), 2)
    with pytest.raises(HgkError, match="dtype"):
        H.moe_route(x.double(), 2)
    with pytest.raises(HgkError, match="GPU"):
        H.moe_route(x, 2)
    y, w = torch.zeros((8, 64), dtype=BF16), torch.zeros((4, 2))
    for a, kw, text in (((y, w.to(BF16)), {}, "weights"), ((y[:7], w), {}, "7 rows"),
                        ((y, w), dict(shared=torch.zeros((4, 63), dtype=BF16)), "shared"),
                        ((y, w), dict(shared=torch.zeros((4, 64))), "shared"),
                        ((y, w), dict(shared_gate=torch.zeros(3)), "shared_gate"),
                        ((y, w), dict(out=torch.zeros((4, 64))), "out"), ((y, w), {}, "GPU")):
        with pytest.raises(HgkError, match=text):
            H.moe_combine(*a, **kw)
    t, n, f, m, c = (torch.zeros(s, dtype=I32) for s in ((3, 4), 3, 9, 1, 3))
    for a, kw, text in (((t.long(), n, f, m, c, 16, 3), {}, "tables"), ((t[0], n, f, m, c, 16, 3), {}, "tables"),
                        ((t.t().contiguous().t(), n, f, m, c, 16, 3), {}, "unit-stride"),
                        ((t, n[:2], f, m, c, 16, 3), {}, "lens"), ((t, n, f, f, c, 16, 3), {}, "n_free"),
                        ((t, n, f.long(), m, c, 16, 3), {}, "free_pages"), ((t, n, f, m, c[:2], 16, 3), {}, "counts"),
                        ((t, n, f, m, c, 16, 3), dict(seqs=c[:2]), "counts"), ((t, n, f, m, c, 0, 3), {}, "page_size"),
                        ((t, n, f, m, c, 16, -1), {}, "tokens"), ((t, n, f, m, c, 16, 3), {}, "GPU")):
        with pytest.raises(HgkError, match=text):
            H.kv_extend(*a, **kw)
    for a, kw, text in (((t, n, f, m, 24), {}, "GPU|page_size"), ((t, n, f, m, 16), dict(keep=c[:2]), "keep"),
                        ((t, n, f, m, 16), dict(owned_from=c[:2]), "owned_from"),
                        ((t, n, f, m, 16), dict(seqs=c.long()), "seqs"), ((t, n, f, m, 16), {}, "GPU")):
        with pytest.raises(HgkError, match=text):
            H.kv_release(*a, **kw)
    p = torch.zeros((4, 16, 2, 64), dtype=BF16)
    q, bt, ln, pt = torch.zeros((2, 4, 64), dtype=BF16), torch.zeros((2, 3), dtype=I32), torch.ones(2, dtype=I32), \
        torch.zeros(2, dtype=I32)
    for a, kw, text in (((q, p, p, bt, ln, pt, 33), {}, "do not hold"), ((q, p, p, bt, ln, pt, -1), {}, "prefix_len"),
                        ((q, p, p, bt, ln, pt, 2 ** 63), {}, "prefix_len"), ((q, p, p, bt, ln, pt.long(), 5), {}, "prefix_table"),
                        ((q, p, p, bt, ln, bt, 5), {}, "prefix_table"), ((q, p, p, bt, ln, pt, 5), dict(window=-1), "window"),
                        ((q, p, p, bt, ln, pt, 5), dict(out=q[:1]), "out"), ((q.float(), p, p, bt, ln, pt, 5), {}, "share"),
                        ((q, p, p, bt, ln, pt, 5), {}, "GPU")):
        with pytest.raises(HgkError, match=text):
            H.shared_prefix_attention(*a, **kw)


def test_shared_prefix_of_a_cache(monkeypatch):
    """The tokens that sequences have on the same pages, and what attend makes of them."""
    monkeypatch.setattr(ops, "kv_copy_pages", lambda *a: None)
    c = H.PagedKVCache(1, 40, 16, 2, 64, device="meta")
    a = c.new()
    c.extend([a], [40])
    assert c.shared_prefix([a]) == 40 and c.shared_prefix([]) == 0
    b = c.fork(a)
    assert c.shared_prefix([a, b]) == 40
    c.extend([a, b], [1, 3])  # the third page is copied for one of them
    assert c.shared_prefix([a, b]) == 32 == c.shared_prefix([b, a])
    d, e = c.fork(a), c.new()
    assert c.shared_prefix([a, d]) == 41 and c.shared_prefix([a, b, d]) == 32
    assert c.shared_prefix([a, e]) == 0
    c.extend([e], [40])
    assert c.shared_prefix([a, e]) == 0
    with pytest.raises(HgkError, match="twice"):
        c.shared_prefix([a, a])
    seen = []
    monkeypatch.setattr(ops, "shared_prefix_attention", lambda q, k, v, t, n, p, m, **kw: seen.append((p.shape, m, kw)))
    from higgs_amd.cache import KVBatch
    kb = KVBatch(torch.zeros((2, 5), dtype=I32), torch.zeros(2, dtype=I32), None)
    c.attend(0, None, kb, prefix=33, window=7)
    assert seen == [(torch.Size([3]), 33, {"q_starts": None, "window": 7})]
