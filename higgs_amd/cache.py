"""The pages of a key-value cache, given out to sequences.

Stands where the reference keeps one growing cache per request
(SteppingKeyValueCache, crates/higgs-models/src/cache.rs:130-312) and clones it
for a shared prompt prefix (crates/higgs-engine/src/prompt_cache.rs:22-307):
here sequences share whole pages, and a fork costs no copy until one of its
branches writes to a page that is only partly filled.

    cache = PagedKVCache(layers, n_pages, page_size, kv_heads, head_dim)
    s = cache.new()
    cache.extend([s], [len(prompt)])               # pages for the prompt
    b = cache.batch([s], [len(prompt)])
    for layer in ...:
        cache.append(layer, k, v, b)
        o = cache.attend(layer, q, b)
    t = cache.fork(s)                              # shares the prompt's pages
    cache.extend([s, t], [1, 1])                   # one new token each
    b = cache.batch([s, t])
"""
from __future__ import annotations

from array import array
from typing import NamedTuple, Optional, Sequence

import numpy as np
import torch

from . import ops
from ._lib import HgkError


class KVBatch(NamedTuple):
    """The device arrays of a call over some sequences' new tokens."""
    block_table: torch.Tensor
    kv_lens: torch.Tensor
    q_starts: Optional[torch.Tensor]


class _Seq:
    __slots__ = ("pages", "length")

    def __init__(self, pages, length):
        self.pages, self.length = pages, length


class PagedKVCache:
    """Pools of key and value pages for every layer ([layers, n_pages,
    page_size, kv_heads, head_dim]) and, on the host, which pages each sequence
    has. Pages are reference counted: fork() shares them, and extend() copies a
    shared page before new tokens go into it. Not for use by several threads at
    once; device work goes to the current stream, so use one stream for all of
    a cache's calls."""

    def __init__(self, layers: int, n_pages: int, page_size: int, kv_heads: int, head_dim: int, *,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if layers < 1 or n_pages < 1:
            raise HgkError(1, f"PagedKVCache: {layers} layers of {n_pages} pages")
        if page_size < 1 or page_size > 65536 or page_size & (page_size - 1):
            raise HgkError(1, f"PagedKVCache: page_size={page_size} must be a power of two in 1..65536")
        if dtype not in (torch.bfloat16, torch.float16) or head_dim not in (64, 96, 128, 256):
            raise HgkError(2, f"PagedKVCache: {dtype} of head_dim {head_dim} (bf16 or f16; 64, 96, 128 or 256)")
        shape = (layers, n_pages, page_size, kv_heads, head_dim)
        self.k_pages = torch.empty(shape, dtype=dtype, device=device)
        self.v_pages = torch.empty(shape, dtype=dtype, device=device)
        self.layers, self.n_pages, self.page_size = layers, n_pages, page_size
        self._refs = [0] * n_pages
        self._free = list(range(n_pages - 1, -1, -1))
        self._seqs: dict[int, _Seq] = {}
        self._next = 0

    # ------------------------------------------------------------ sequences
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _seq(self, seq: int) -> _Seq:
        try:
            return self._seqs[seq]
        except KeyError:
            raise HgkError(1, f"PagedKVCache: no sequence {seq}") from None

    def _several(self, seqs: Sequence[int], counts: Optional[Sequence[int]]):
        if counts is not None and len(counts) != len(seqs):
            raise HgkError(1, f"PagedKVCache: {len(counts)} counts for {len(seqs)} sequences")
        if len(set(seqs)) != len(seqs):
            raise HgkError(1, "PagedKVCache: a sequence is named twice")
        if counts is not None and any(c < 0 for c in counts):
            raise HgkError(1, "PagedKVCache: counts must not be negative")
        return [self._seq(s) for s in seqs]

    def new(self) -> int:
        """An empty sequence's handle."""
        self._seqs[self._next] = _Seq(array("i"), 0)
        self._next += 1
        return self._next - 1

    def length(self, seq: int) -> int:
        return self._seq(seq).length

    def pages(self, seq: int) -> list:
        """The sequence's pages in order (-1: trimmed)."""
        return list(self._seq(seq).pages)

    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens, on the same pages."""
        s = self._seq(seq)
        for p in s.pages:
            if p >= 0:
                self._refs[p] += 1
        f = self.new()
        self._seqs[f] = _Seq(array("i", s.pages), s.length)
        return f

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            self._free.append(page)

    def free(self, seq: int) -> None:
        """Ends a sequence; pages that no other sequence has are free again."""
        s = self._seq(seq)
        del self._seqs[seq]
        for p in s.pages:
            if p >= 0:
                self._drop(p)

    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> None:
        """Room for counts[i] more tokens of seqs[i]: pages are given out, and
        a shared, partly filled last page is copied in every layer. Raises
        HgkError, with nothing changed, when there are not enough free pages."""
        found = self._several(seqs, counts)
        ps, refs, copies, need = self.page_size, {}, [], 0
        for s, n in zip(found, counts):
            if s.length + n > 2 ** 30:  # what a call's table may hold
                raise HgkError(1, "PagedKVCache: a sequence of more than 2^30 tokens")
            if n and s.length % ps:
                last = s.pages[-1]
                shared = refs.get(last, self._refs[last])
                if shared > 1:
                    refs[last] = shared - 1
                    copies.append(s)
            need += -(-(s.length + n) // ps) - len(s.pages)
        if need + len(copies) > len(self._free):
            raise HgkError(1, f"PagedKVCache: {need + len(copies)} pages needed, {len(self._free)} free")
        if copies:
            dst = self._free[:-len(copies) - 1:-1]
            ops.kv_copy_pages(self.k_pages, self.v_pages, [s.pages[-1] for s in copies], dst)
            del self._free[-len(copies):]
            for s, p in zip(copies, dst):
                self._drop(s.pages[-1])  # still held by another sequence
                self._refs[p] = 1
                s.pages[-1] = p
        for s, n in zip(found, counts):
            s.length += n
            while len(s.pages) * ps < s.length:
                p = self._free.pop()
                self._refs[p] = 1
                s.pages.append(p)

    def trim(self, seq: int, window: int, sinks: int = 0) -> int:
        """Gives up the pages that a query at the sequence's last position, or
        a later one, does not see under ``window`` and ``sinks``; calls over
        the sequence then have to use them (or a smaller window). Returns how
        many pages were given up."""
        s = self._seq(seq)
        if window < 1 or sinks < 0:
            raise HgkError(1, f"PagedKVCache: window={window}, sinks={sinks}")
        ps, dropped = self.page_size, 0
        for e in range(-(-sinks // ps), max(0, s.length - window) // ps):
            if s.pages[e] >= 0:
                self._drop(s.pages[e])
                s.pages[e] = -1
                dropped += 1
        return dropped

    def compact(self) -> int:
        """Moves the pages in use to the lowest indices and returns how many
        were moved. Block tables made before no longer hold."""
        live = self.n_pages - len(self._free)
        src = [p for p in range(live, self.n_pages) if self._refs[p]]
        if src:
            dst = [p for p in range(live) if not self._refs[p]]
            ops.kv_copy_pages(self.k_pages, self.v_pages, src, dst)
            to = dict(zip(src, dst))
            for s, d in to.items():
                self._refs[d], self._refs[s] = self._refs[s], 0
            for s in self._seqs.values():
                s.pages = array("i", [to.get(p, p) for p in s.pages])
        self._free = list(range(self.n_pages - 1, live - 1, -1))
        return len(src)

    # ------------------------------------------------------------ device calls
    def batch(self, seqs: Sequence[int], counts: Optional[Sequence[int]] = None) -> KVBatch:
        """Table, lengths and starts of a call over the last counts[i] tokens
        of each sequence (without counts: the last one of each). Holds until a
        sequence in it is extended, trimmed or freed, or the pool compacted."""
        found = self._several(seqs, counts)
        for i, s in enumerate(found):
            if s.length < (1 if counts is None else counts[i]):
                raise HgkError(1, f"PagedKVCache: sequence {seqs[i]} has {s.length} tokens")
        table = np.full((len(found), max((len(s.pages) for s in found), default=0)), -1, np.int32)
        for row, s in zip(table, found):
            row[:len(s.pages)] = s.pages
        dev = self.k_pages.device
        lens = torch.tensor([s.length for s in found], dtype=torch.int32, device=dev)
        starts = None
        if counts is not None:
            starts = torch.from_numpy(np.cumsum([0, *counts]).astype(np.int32)).to(dev)
        return KVBatch(torch.from_numpy(table).to(dev), lens, starts)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, batch: KVBatch) -> None:
        """kv_append of one layer's keys and values."""
        ops.kv_append(k, v, self.k_pages[layer], self.v_pages[layer], batch.block_table,
                      batch.kv_lens, q_starts=batch.q_starts)

    def attend(self, layer: int, q: torch.Tensor, batch: KVBatch, **kw) -> torch.Tensor:
        """paged_attention over one layer's pages (scale, window, sinks,
        softcap, out as there)."""
        return ops.paged_attention(q, self.k_pages[layer], self.v_pages[layer], batch.block_table,
                                   batch.kv_lens, q_starts=batch.q_starts, **kw)
