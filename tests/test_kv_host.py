"""The paged key-value cache without a GPU: the C ABI's layout and refusals,
the kernels' index arithmetic compiled for the host, and PagedKVCache's page
bookkeeping (with the page copy done by torch)."""
from __future__ import annotations

import ctypes as C
import os
import random
import shutil
import subprocess

import pytest
import torch

import higgs_amd as H
from higgs_amd import _lib, ops
from higgs_amd._lib import HgkError, HgkKvBatch, HgkKvPages

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20  # never dereferenced: such calls end in the checks, or have nothing to do


def pages(**kw):
    d = dict(dtype=1, page_size=16, n_pages=8, kv_heads=2, head_dim=64, k=FAKE, v=FAKE,
             k_strides=(C.c_int64 * 3)(2048, 128, 64), v_strides=(C.c_int64 * 3)(2048, 128, 64))
    return HgkKvPages(**{**d, **kw})


def batch(**kw):
    d = dict(batch=2, tokens=2, block_table=FAKE, table_stride=4, table_width=4, kv_lens=FAKE,
             q_starts=None)
    return HgkKvBatch(**{**d, **kw})


def st(*v):
    return (C.c_int64 * len(v))(*v)


def attention(p=None, b=None, q=FAKE, qs=(256, 64), heads=4, scale=0.125, softcap=0.0, window=0, sinks=0,
              out=FAKE, os_=(256, 64), ws=None, ws_bytes=0):
    L = _lib.lib()
    s = L.hgk_paged_attention(C.byref(p or pages()), C.byref(b or batch()), q, st(*qs), heads, scale, softcap,
                              window, sinks, out, st(*os_), ws, ws_bytes, None)
    return s, L.hgk_last_error().decode()


def test_struct_layouts():
    """ctypes, the packed form the Python calls use, and the C header agree."""
    import struct

    assert C.sizeof(HgkKvPages) == ops._KV_PAGES.size and C.sizeof(HgkKvBatch) == ops._KV_BATCH.size
    got = HgkKvPages.from_buffer_copy(ops._KV_PAGES.pack(1, 16, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13))
    assert (got.dtype, got.page_size, got.n_pages, got.kv_heads, got.head_dim, got.k, list(got.k_strides),
            got.v, list(got.v_strides)) == (1, 16, 3, 4, 5, 6, [7, 8, 9], 10, [11, 12, 13])
    got = HgkKvBatch.from_buffer_copy(ops._KV_BATCH.pack(1, 2, 3, 4, 5, 6, 7))
    assert [getattr(got, f[0]) for f in HgkKvBatch._fields_] == [1, 2, 3, 4, 5, 6, 7]
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc:
        import tempfile

        src = "#include <stdio.h>\n#include <stddef.h>\n#include \"higgs_hip.h\"\nint main(void){"
        want = []
        for name, cls in (("hgk_kv_pages", HgkKvPages), ("hgk_kv_batch", HgkKvBatch)):
            src += f"printf(\"%zu \", sizeof({name}));"
            want.append(C.sizeof(cls))
            for f in cls._fields_:
                src += f"printf(\"%zu \", offsetof({name}, {f[0]}));"
                want.append(getattr(cls, f[0]).offset)
        with tempfile.TemporaryDirectory() as d:
            open(os.path.join(d, "l.c"), "w").write(src + "return 0;}\n")
            subprocess.run([cc, "-I", os.path.join(ROOT, "include"), os.path.join(d, "l.c"), "-o",
                            os.path.join(d, "l")], check=True)
            out = subprocess.run([os.path.join(d, "l")], capture_output=True, text=True, check=True).stdout
        assert [int(v) for v in out.split()] == want


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=0), 2, "bf16 or f16"), (dict(dtype=9), 2, "dtype"), (dict(page_size=0), 1, "page_size"),
    (dict(page_size=24), 1, "page_size"), (dict(page_size=1 << 17), 1, "page_size"),
    (dict(n_pages=-1), 1, "n_pages"), (dict(n_pages=1 << 31), 1, "n_pages"), (dict(kv_heads=0), 1, "kv_heads"),
    (dict(head_dim=80), 2, "head_dim"), (dict(k=None), 1, "null"), (dict(v=FAKE + 2), 1, "aligned"),
    (dict(k_strides=st(2048, 128, 60)), 1, "multiples of 8"), (dict(v_strides=st(-2048, 128, 64)), 1, "multiples of 8"),
])
def test_refused_pages(kw, status, text):
    p, L = pages(**kw), _lib.lib()
    assert attention(p=p) == (status, L.hgk_last_error().decode()) and text in L.hgk_last_error().decode()
    assert L.hgk_paged_attention_workspace(C.byref(p), C.byref(batch()), 4, 0, 0) in (-1, 0)
    s = L.hgk_kv_append(C.byref(p), C.byref(batch()), FAKE, st(128, 64), FAKE, st(128, 64), None)
    assert s == status and text in L.hgk_last_error().decode()
    one = (C.c_int32 * 1)(0), (C.c_int32 * 1)(1)
    s = L.hgk_kv_copy_pages(C.byref(p), 1, None, *one, 1, None)
    assert s == status or kw.get("n_pages") == -1
    assert text in L.hgk_last_error().decode()


@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1, tokens=-1), "out of range"), (dict(tokens=-1, q_starts=FAKE), "out of range"),
    (dict(tokens=3), "3 rows for 2"), (dict(table_width=1 << 27), "too wide"), (dict(table_width=-1), "table"), (dict(table_stride=-4), "table"),
    (dict(kv_lens=None), "null"), (dict(block_table=None), "null"), (dict(tokens=1 << 31, q_starts=FAKE), "out of range"),
])
def test_refused_batches(kw, text):
    L, b = _lib.lib(), batch(**kw)
    s, msg = attention(b=b)
    assert s == 1 and text in msg
    s = L.hgk_kv_append(C.byref(pages()), C.byref(b), FAKE, st(128, 64), FAKE, st(128, 64), None)
    assert s == 1 and text in L.hgk_last_error().decode()


def test_refused_attention_arguments():
    for kw, text in ((dict(heads=0), "heads"), (dict(heads=3), "heads"), (dict(window=-1), "window"),
                     (dict(sinks=-1), "sinks"), (dict(scale=float("nan")), "scale"),
                     (dict(scale=float("inf")), "scale"), (dict(softcap=-1.0), "softcap"),
                     (dict(softcap=float("nan")), "softcap"), (dict(softcap=float("inf")), "softcap"),
                     (dict(q=None), "null q"), (dict(out=None), "null out"), (dict(q=FAKE + 8), "aligned"),
                     (dict(qs=(256, 60)), "multiples"), (dict(os_=(256, -64)), "multiples"),
                     (dict(os_=(0, 64)), "overlap"), (dict(os_=(256, 56)), "overlap"),
                     (dict(os_=(64, 64)), "overlap"), (dict(os_=(192, 64)), "overlap")):
        s, msg = attention(**kw)
        assert s == 1 and text in msg, (kw, msg)
    L = _lib.lib()
    assert L.hgk_paged_attention_workspace(C.byref(pages()), C.byref(batch()), 3, 0, 0) == -1
    assert L.hgk_paged_attention_workspace(None, C.byref(batch()), 4, 0, 0) == -1
    assert L.hgk_paged_attention_workspace(C.byref(pages()), None, 4, 0, 0) == -1
    # a workspace that is asked for and missing, short or unaligned
    long = batch(batch=1, tokens=1, table_width=1 << 16, table_stride=1 << 16)
    need = L.hgk_paged_attention_workspace(C.byref(pages()), C.byref(long), 4, 0, 0)
    if need > 0:
        for ws, n in ((None, need), (FAKE, need - 1), (FAKE + 4, need)):
            s, msg = attention(b=long, ws=ws, ws_bytes=n)
            assert s == 1 and "workspace" in msg
    for b in (batch(batch=0, tokens=0), batch(batch=3, tokens=0, q_starts=FAKE),
              batch(batch=0, tokens=9, q_starts=FAKE)):
        assert L.hgk_paged_attention_workspace(C.byref(pages()), C.byref(b), 4, 0, 0) == 0
        assert attention(b=b, q=None, out=None)[0] == 0
    # nothing to do: no launch, and no data needed
    none = batch(batch=0, tokens=0, block_table=None, kv_lens=None)
    assert attention(b=none, q=None, out=None)[0] == 0
    assert L.hgk_kv_append(C.byref(pages()), C.byref(none), None, None, None, None, None) == 0
    rows = batch(batch=0, tokens=5, q_starts=FAKE)
    assert attention(b=rows, q=None, out=None)[0] == 0


def test_refused_copies():
    L = _lib.lib()

    def copy(src, dst, layers=1, strides=None, **kw):
        s = L.hgk_kv_copy_pages(C.byref(pages(**kw)), layers, strides, (C.c_int32 * len(src))(*src),
                                (C.c_int32 * len(dst))(*dst), len(src), None)
        return s, L.hgk_last_error().decode()

    for src, dst, text in (([0], [8], "outside"), ([8], [0], "outside"), ([-1], [0], "outside"),
                           ([0], [-1], "outside"), ([0, 1], [2, 2], "twice"), ([0, 2], [2, 3], "source"),
                           ([3], [3], "source")):
        s, msg = copy(src, dst)
        assert s == 1 and text in msg, msg
    assert copy([0], [1], layers=-1)[0] == 1 and copy([0], [1], layers=2)[0] == 1
    assert copy([0], [1], layers=2, strides=st(60, 64))[0] == 1
    assert "overlap" in copy([0], [1], layers=2, strides=st(0, 1 << 20))[1]
    for lk, lv in ((64, 1 << 20), (1 << 20, 8192), (2048, 1 << 20)):  # layers inside each other
        assert "overlap" in copy([0], [1], layers=2, strides=st(lk, lv))[1], (lk, lv)
    for k in ((0, 128, 64), (2048, 128, 56), (2048, 64, 64), (1024, 128, 64), (2048, 64, 512)):
        assert "overlap" in copy([0], [1], k_strides=st(*k))[1], k
    for k in ((2048, 128, 64), (2048, 64, 1024), (64, 1024, 512), (64, 512, 8192)):  # any order of the axes
        assert L.hgk_kv_append(C.byref(pages(v_strides=st(*k))), C.byref(batch()), None, st(128, 64), FAKE,
                               st(128, 64), None) == 1 and "null k" in L.hgk_last_error().decode(), k
    assert copy([], []) == (0, "") and copy([0], [1], layers=0)[0] == 0


def test_refusals_of_the_python_calls():
    """Checked before any device work, so CPU tensors show them."""
    p = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    t, n = torch.zeros((2, 3), dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    bad = [
        lambda: H.paged_attention(q, p, p[:, :, :1], t, n), lambda: H.paged_attention(q, p, p.half(), t, n),
        lambda: H.paged_attention(q[..., :32], p, p, t, n), lambda: H.paged_attention(q.half(), p, p, t, n),
        lambda: H.paged_attention(q, p, p, t.long(), n), lambda: H.paged_attention(q, p, p, t, n.long()),
        lambda: H.paged_attention(q, p, p, t, n[:1]), lambda: H.paged_attention(q, p, p, t[0], n),
        lambda: H.paged_attention(q, p, p, t, n, q_starts=n), lambda: H.paged_attention(q, p, p, t, n, out=q[:1]),
        lambda: H.paged_attention(q, p, p, t, n, out=q.float()),
        lambda: H.paged_attention(q.transpose(1, 2), p, p, t, n), lambda: H.paged_attention(q, p[0], p[0], t, n),
        lambda: H.kv_append(k, k[:1], p, p, t, n), lambda: H.kv_append(k[:, :1], k[:, :1], p, p, t, n),
        lambda: H.kv_append(k.float(), k, p, p, t, n), lambda: H.kv_copy_pages(p, p, [0], [1, 2]),
        lambda: H.kv_copy_pages(p, p, [0], [2 ** 32 + 1]), lambda: H.paged_attention(q, p, p, t, n, window=2 ** 64),
        lambda: H.paged_attention(q, p, p, t, n, sinks=-1), lambda: H.kv_copy_pages(p, p, [0.5], [1]),
        # nothing of this is on a GPU
        lambda: H.paged_attention(q, p, p, t, n), lambda: H.kv_append(k, k, p, p, t, n),
        lambda: H.kv_copy_pages(p, p, [0], [1]),
    ]
    for f in bad:
        with pytest.raises(HgkError):
            f()


# ---------------------------------------------------------------- index arithmetic
CHECK = r"""
#include "kv.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
using namespace hgk;
#define MUST(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
  // what the arrays may hold when a caller's own bookkeeping is wrong
  const int32_t odd[] = {0, 1, 2, 3, 5, 7, 8, 9, -1, -2147483647 - 1, 2147483647, 100, 6, 4};
  const int n_odd = sizeof odd / sizeof *odd;
  srand(1);
  for (int it = 0; it < 200000; ++it) {
    const int batch = 1 + rand() % 5, tokens = rand() % 9, width = rand() % 4;
    std::vector<int32_t> starts(batch + 1), lens(batch), table((size_t)batch * width + 1, 12345);
    for (auto& v : starts) v = odd[rand() % n_odd];
    for (auto& v : lens) v = odd[rand() % n_odd];
    for (int i = 0; i < batch * width; ++i) table[i] = odd[rand() % n_odd];
    KvBatchView b{table.data(), lens.data(), rand() % 3 ? starts.data() : nullptr, width, width, batch,
                  tokens};
    if (!b.starts) b.tokens = batch;
    KvView p{};
    p.n_pages = rand() % 9;
    p.page_shift = rand() % 4;
    p.page_mask = (1 << p.page_shift) - 1;
    for (int s = 0; s < batch; ++s) {
      const KvSeq q = kv_seq(b, s);
      MUST(q.n >= 0 && q.first >= 0 && (int64_t)q.first + q.n <= b.tokens);
      for (int k = 0; k < 6; ++k) {
        const int32_t pos = k == 5 ? 2147483647 : (rand() % 40);
        const int32_t page = kv_page(p, b, s, pos);
        MUST(page == -1 || (page >= 0 && page < p.n_pages));
        const int e = pos >> p.page_shift;
        if (e < width && table[(size_t)s * width + e] >= 0 && table[(size_t)s * width + e] < p.n_pages)
          MUST(page == table[(size_t)s * width + e]);
        else
          MUST(page == -1);
      }
    }
    for (int t = 0; t < b.tokens; ++t) {
      const int s = kv_row_owner(b, t);
      MUST(s >= 0 && s < batch);
    }
    // in order: every row finds its sequence
    starts[0] = 0;
    for (int s = 0; s < batch; ++s) starts[s + 1] = starts[s] + rand() % 3;
    b.starts = starts.data();
    b.tokens = starts[batch] + 2;
    for (int s = 0; s < batch; ++s)
      for (int t = starts[s]; t < starts[s + 1]; ++t) MUST(kv_row_owner(b, t) == s);
  }
  printf("ok\n");
  return 0;
}
"""


def test_bad_metadata_reaches_no_memory(tmp_path):
    """kv_seq, kv_page and kv_row_owner, which every kernel goes through,
    compiled for the host and run over metadata that is out of order and out
    of range; every array is exactly as long as the call says (and checked by
    the host's address sanitizer)."""
    from higgs_amd import build

    src = tmp_path / "check.cpp"
    src.write_text(CHECK)
    exe = tmp_path / "check"
    cc = build.hipcc()
    subprocess.run([cc, "-x", "hip", "--offload-host-only", "-nogpulib", "-std=c++17", "-O1", "-w",
                    "-Xarch_host", "-fsanitize=address", "-I", os.path.join(ROOT, "higgs_amd", "csrc"),
                    str(src), "-o", str(exe)], check=True, capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120,
                       env={**os.environ, "ASAN_OPTIONS": "detect_leaks=0"})
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


# ---------------------------------------------------------------- bookkeeping
def torch_copy(k, v, src, dst):
    assert len(set(dst)) == len(dst) and not set(dst) & set(src)
    for t in (k, v):
        t[:, dst] = t[:, src]


@pytest.fixture
def cpu_copies(monkeypatch):
    monkeypatch.setattr(ops, "kv_copy_pages", torch_copy)


def small(n_pages=12, page=4):
    return H.PagedKVCache(2, n_pages, page, 1, 64, dtype=torch.float16, device="cpu")


def test_pages_are_shared_and_copied_on_write(cpu_copies):
    c = small()
    a = c.new()
    c.extend([a], [6])
    assert c.length(a) == 6 and len(c.pages(a)) == 2 and c.free_pages == 10
    b, d = c.fork(a), c.fork(a)
    assert c.pages(b) == c.pages(a) and c.free_pages == 10
    for p in c.pages(a):
        c.k_pages[:, p] = p + 1
    c.extend([b, a, d], [1, 1, 0])  # both write to the shared half page; d holds on to it
    assert c.free_pages == 8 and len({c.pages(s)[1] for s in (a, b, d)}) == 3
    assert c.pages(a)[0] == c.pages(b)[0] == c.pages(d)[0]
    for s in (a, b):
        assert (c.k_pages[:, c.pages(s)[1]] == c.pages(d)[1] + 1).all()
    last = c.pages(d)[1]
    c.extend([d], [1])  # its own by now
    assert c.pages(d)[1] == last and c.free_pages == 8
    c.free(a)
    c.free(b)
    c.free(d)
    assert c.free_pages == 12


def test_full_pages_are_not_copied(cpu_copies):
    c = small()
    a = c.new()
    c.extend([a], [8])
    b = c.fork(a)
    c.extend([a, b], [1, 1])
    assert c.pages(a)[:2] == c.pages(b)[:2] and c.pages(a)[2] != c.pages(b)[2] and c.free_pages == 8


def test_running_out_changes_nothing(cpu_copies):
    c = small(n_pages=3)
    a = c.new()
    c.extend([a], [6])
    b = c.fork(a)
    before = (c.pages(a), c.pages(b), c.free_pages, c.length(a))
    with pytest.raises(HgkError, match="free"):
        c.extend([a, b], [3, 1])
    assert before == (c.pages(a), c.pages(b), c.free_pages, c.length(a))
    c.extend([a, b], [1, 1])
    assert c.free_pages == 0


def test_refused_sequences(cpu_copies):
    c = small()
    a = c.new()
    for f in (lambda: c.length(7), lambda: c.fork(7), lambda: c.free(7), lambda: c.extend([a, a], [1, 1]),
              lambda: c.extend([a], [-1]), lambda: c.extend([a], [1, 2]), lambda: c.batch([a]),
              lambda: c.batch([a, a], [0, 0]), lambda: c.batch([a], [1]), lambda: c.trim(a, 0),
              lambda: c.trim(a, 4, -1), lambda: c.extend([a], [2 ** 31])):
        with pytest.raises(HgkError):
            f()
    c.free(a)
    with pytest.raises(HgkError):
        c.free(a)
    for kw in ((0, 4, 4), (2, 0, 4), (2, 4, 3), (2, 4, 0)):
        with pytest.raises(HgkError):
            H.PagedKVCache(*kw, 1, 64, device="cpu")
    for kw in ({"dtype": torch.float32}, {"head_dim": 80}):
        with pytest.raises(HgkError):
            H.PagedKVCache(2, 4, 4, 1, **{"head_dim": 64, "device": "cpu", **kw})


def test_batches(cpu_copies):
    c = small()
    a, b = c.new(), c.new()
    c.extend([a, b], [5, 9])
    t = c.batch([b, a])
    assert t.q_starts is None and t.kv_lens.tolist() == [9, 5]
    assert t.block_table.tolist() == [c.pages(b), [*c.pages(a), -1]]
    t = c.batch([a, b], [2, 0])
    assert t.q_starts.tolist() == [0, 2, 2] and t.kv_lens.dtype == t.q_starts.dtype == torch.int32
    t = c.batch([], [])
    assert t.block_table.shape == (0, 0) and t.q_starts.tolist() == [0]


def test_trim_keeps_what_is_seen(cpu_copies):
    """For every length, window and number of sinks: a page is given up only
    when no query from the last position on sees a token of it, and always then."""
    for length in range(1, 30):
        for window in (1, 2, 4, 5, 9, 40):
            for sinks in (0, 1, 4, 5, 50):
                c = small()
                s = c.new()
                c.extend([s], [length])
                c.trim(s, window, sinks)
                for e, p in enumerate(c.pages(s)):
                    tokens = range(4 * e, 4 * e + 4)
                    seen = any(j < sinks or j > (length - 1) - window for j in tokens)
                    assert (p >= 0) == seen, (length, window, sinks, e)
                assert c.free_pages == 12 - sum(p >= 0 for p in c.pages(s))
                c.free(s)
                assert c.free_pages == 12


def test_random_use_keeps_every_sequences_tokens(cpu_copies):
    """Extends, forks, trims, frees and compactions in random order against a
    list of each sequence's tokens; pages are used by whom their counts say."""
    rng = random.Random(3)
    c = small(n_pages=40)
    want, stamp = {}, 0
    for _ in range(1500):
        what = rng.choice(["new", "extend", "extend", "extend", "fork", "free", "compact", "trim"])
        live = list(want)
        if what == "new" and len(live) < 6:
            want[c.new()] = []
        elif what == "extend" and live:
            seqs = rng.sample(live, rng.randint(1, len(live)))
            counts = [rng.randint(0, 5) for _ in seqs]
            try:
                c.extend(seqs, counts)
            except HgkError:
                continue
            for s, n in zip(seqs, counts):
                for i in range(n):
                    stamp += 1
                    want[s].append(stamp % 2000)
                    pos = len(want[s]) - 1
                    c.k_pages[:, c.pages(s)[pos // 4], pos % 4] = want[s][-1]
        elif what == "fork" and live and len(live) < 6:
            s = rng.choice(live)
            want[c.fork(s)] = list(want[s])
        elif what == "free" and live:
            s = rng.choice(live)
            c.free(s)
            del want[s]
        elif what == "compact":
            c.compact()
            used = {p for s in want for p in c.pages(s) if p >= 0}
            assert used == set(range(len(used)))
        elif what == "trim" and live:
            s = rng.choice(live)
            if want[s]:
                c.trim(s, rng.randint(1, 20), rng.randint(0, 6))
        counts = {}
        for s in want:
            assert c.length(s) == len(want[s]) and len(c.pages(s)) == -(-len(want[s]) // 4)
            for e, p in enumerate(c.pages(s)):
                if p >= 0:
                    counts[p] = counts.get(p, 0) + 1
                    part = want[s][4 * e:4 * e + 4]
                    assert c.k_pages[1, p, :len(part), 0, 0].tolist() == part
        assert c.free_pages == 40 - len(counts)
        assert all(c._refs[p] == counts.get(p, 0) for p in range(40))
