"""PagedKVCache.attend refuses a prefix that the batch's sequences do not share."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
from higgs_amd import HgkError, ops
from higgs_amd.cache import KVBatch


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(ops, "kv_copy_pages", lambda *a: None)
    calls = []
    monkeypatch.setattr(ops, "shared_prefix_attention", lambda q, k, v, t, n, p, m, **kw: calls.append((p.tolist(), m)))
    c = H.PagedKVCache(1, 60, 16, 2, 64, device="cpu")
    c.calls = calls
    return c


def test_prefix_past_what_is_shared(cache):
    c = cache
    a = c.new()
    c.extend([a], [40])
    b = c.fork(a)
    whole = c.batch([a, b])
    c.attend(0, None, whole, prefix=40)
    c.extend([a, b], [1, 3])  # the third page is copied for one of them
    both = c.batch([a, b])
    for n in (1, 31, 32):
        c.attend(0, None, both, prefix=n)
    for n in (33, 40, 41, 10 ** 6):
        with pytest.raises(HgkError, match="share 32 tokens"):
            c.attend(0, None, both, prefix=n)
    assert c.calls == [(c.pages(a)[:2] + [whole.block_table[0, 2].item()], 40), (c.pages(a)[:1], 1), (c.pages(a)[:2], 31),
                       (c.pages(a)[:2], 32)]


def test_prefix_of_strangers_and_of_one(cache):
    c = cache
    a, b = c.new(), c.new()
    c.extend([a, b], [40, 70])
    with pytest.raises(HgkError, match="share 0 tokens"):
        c.attend(0, None, c.batch([a, b]), prefix=1)
    c.attend(0, None, c.batch([b]), prefix=70)
    with pytest.raises(HgkError, match="share 70 tokens"):
        c.attend(0, None, c.batch([b], [5]), prefix=71)
    with pytest.raises(HgkError, match="share 0 tokens"):
        c.attend(0, None, c.batch([]), prefix=1)


def test_prefix_after_a_trim(cache):
    """Pages that one of them has given up are no longer shared."""
    c = cache
    a = c.new()
    c.extend([a], [128])
    b = c.fork(a)
    c.extend([b], [400])
    c.trim(b, 100, sinks=16)
    with pytest.raises(HgkError, match="share 16 tokens"):
        c.attend(0, None, c.batch([a, b]), prefix=17)
    c.trim(a, 20, sinks=16)
    assert c.shared_prefix([a, b]) == c.batch([a, b]).shared(16) == 96
    c.attend(0, None, c.batch([a, b]), prefix=96)


def test_batches_are_what_they_were(cache):
    c = cache
    a, b = c.new(), c.new()
    c.extend([a, b], [40, 7])
    batch = c.batch([a, b])
    table, lens, starts = batch
    assert isinstance(batch, KVBatch) and starts is None and torch.equal(lens, torch.tensor([40, 7], dtype=torch.int32))
    assert table.tolist() == [c.pages(a), c.pages(b) + [-1, -1]]
    # a batch made otherwise is the caller's own affair
    c.attend(0, None, KVBatch(table, lens, None), prefix=33)
    c.attend(0, None, batch._replace(kv_lens=lens + 1), prefix=33)
    assert len(c.calls) == 2
