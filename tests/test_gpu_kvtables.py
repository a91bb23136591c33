"""kv_extend, kv_release and kv_append by slots against a model of them on the
host, number by number."""
from __future__ import annotations

import random

import pytest
import torch

import higgs_amd as H
import kv_ref as R

pytestmark = pytest.mark.gpu

I32 = torch.int32


class Model:
    """The state, with the calls' results worked out one token after the other."""

    def __init__(self, seed, rows, width, page, n_pages, lens):
        self.rng = random.Random(seed)
        self.rows, self.width, self.page, self.n_pages = rows, width, page, n_pages
        order = list(range(n_pages))
        self.rng.shuffle(order)
        self.stack, self.lens = order, list(lens)
        self.tables = [[-7] * width for _ in range(rows)]
        for r, n in enumerate(lens):
            for e in range(-(-n // page)):
                self.tables[r][e] = self.stack.pop()
        self.behind = []  # what lies on the stack behind its free entries

    def state(self, dev):
        t = lambda v: torch.tensor(v, dtype=I32, device=dev)
        free = self.stack + [0] * (self.n_pages - len(self.stack))
        return (t(self.tables).reshape(self.rows, self.width), t(self.lens), t(free), t([len(self.stack)]))

    def status(self, seqs, counts, tokens):
        st, need, seen = 0, 0, set()
        for s, c in zip(seqs, counts):
            if not 0 <= s < self.rows or s in seen or c < 0:
                st |= 4
            seen.add(s)
            if 0 <= s < self.rows:
                now = self.lens[s] + max(c, 0)
                if -(-now // self.page) > self.width:
                    st |= 2
                need += -(-now // self.page) - -(-self.lens[s] // self.page)
        if need > len(self.stack):
            st |= 1
        if sum(max(c, 0) for s, c in zip(seqs, counts) if 0 <= s < self.rows) > tokens:
            st |= 8
        return st

    def extend(self, seqs, counts, tokens):
        st = self.status(seqs, counts, tokens)
        if st:
            counts = [0] * len(seqs)
        slots, positions, starts = [], [], [0]
        for s, c in zip(seqs, counts):
            for p in range(self.lens[s] if c else 0, (self.lens[s] + c) if c else 0):
                if p % self.page == 0:
                    self.tables[s][p // self.page] = self.stack.pop()
                slots.append(self.tables[s][p // self.page] * self.page + p % self.page)
                positions.append(p)
            if c:
                self.lens[s] += c
            starts.append(len(slots))
        kv = [self.lens[s] if 0 <= s < self.rows else 0 for s in seqs]
        pad = tokens - len(slots)
        return st, kv, starts, slots + [-1] * pad, positions + [0] * pad

    def block_table(self, seqs):
        out = []
        for s in seqs:
            n = -(-self.lens[s] // self.page) if 0 <= s < self.rows else 0
            n = min(n, self.width)
            out.append((self.tables[s][:n] if n else []) + [-1] * (self.width - n))
        return out

    def release(self, seqs, keep, owned=None):
        for s, k in zip(seqs, keep):
            k = min(max(k, 0), self.lens[s])
            first = max(-(-k // self.page), 0 if owned is None else owned[s])
            self.stack += self.tables[s][first:-(-self.lens[s] // self.page)]
            self.lens[s] = k


def check_state(m, tables, lens, free, n_free):
    assert lens.tolist() == m.lens and n_free.tolist() == [len(m.stack)]
    assert free.tolist()[:len(m.stack)] == m.stack
    assert tables.tolist() == m.tables


def check_step(m, step, seqs, want, all_rows):
    st, kv, starts, slots, positions = want
    assert step.status.tolist() == [st]
    assert step.kv_lens.tolist() == kv and step.q_starts.tolist() == starts
    assert step.slots.tolist() == slots and step.positions.tolist() == positions
    assert step.slots.dtype == torch.int64
    if not all_rows:
        assert step.block_table.tolist() == m.block_table(seqs)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("page", [1, 4, 16, 256])
@pytest.mark.parametrize("rows,batch", [(1, 1), (5, 5), (70, 33), (1100, 1100), (1500, 1300)])
def test_steps(dev, rows, batch, page, inplace):
    """Extends of some and of all rows, ends and rollbacks, one after the other."""
    rng = random.Random(rows + page)
    lens = [rng.choice([0, 1, page - 1, page, page + 1, 3 * page + 2]) for _ in range(rows)]
    m = Model(rows, rows, 12, page, rows * 12 + 3, lens)
    state = m.state(dev)
    for step in range(4):
        seqs = rng.sample(range(rows), batch)
        some = batch < rows or step % 2 == 0
        if not some:
            seqs = list(range(rows))
        some_counts = [0, 1, 2] + ([page, 2 * page + 1] if rows * page < 20000 else [])
        counts = [1] * batch if step == 1 else [rng.choice(some_counts) for _ in seqs]
        counts = [min(c, 12 * page - m.lens[s]) for s, c in zip(seqs, counts)]
        tokens = sum(counts) + rng.choice([0, 1, 300])
        s = H.kv_extend(*state, torch.tensor(counts, dtype=I32, device=dev), page, tokens, inplace=inplace,
                        seqs=torch.tensor(seqs, dtype=I32, device=dev) if some else None)
        check_step(m, s, seqs, m.extend(seqs, counts, tokens), not some)
        assert (s.lens is state[1]) == inplace and (s.n_free is state[3]) == inplace
        assert some or s.block_table is state[0]
        state = (state[0], s.lens, state[2], s.n_free)
        check_state(m, *state)
        ends = rng.sample(range(rows), (batch + 1) // 2)
        keep = [rng.choice([0, 0, m.lens[e], m.lens[e] - 1, m.lens[e] + 5, -3, m.lens[e] // 2]) for e in ends]
        r = H.kv_release(*state, page, seqs=torch.tensor(ends, dtype=I32, device=dev), inplace=inplace,
                         keep=torch.tensor(keep, dtype=I32, device=dev))
        m.release(ends, keep)
        assert r.status.tolist() == [0] and (r.lens is state[1]) == inplace
        state = (state[0], r.lens, state[2], r.n_free)
        check_state(m, *state)
    r = H.kv_release(*state, page, inplace=inplace)
    m.release(range(rows), [0] * rows)
    check_state(m, state[0], r.lens, state[2], r.n_free)
    assert sorted(m.stack) == list(range(m.n_pages))


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("seqs,counts,tokens,free,status", [
    ([0, 1, 2], [5, 4, 1], 10, 2, 1),          # three pages of two
    ([0, 1, 2], [5, 5, 1], 11, 3, 1),
    ([0, 1, 2], [5, 4, 1], 9, 9, 8),
    ([0, 1, 2], [30, 4, 1], 99, 9, 3),         # 9 pages of a width of 8: 8 + 1 + 1 new ones of 9
    ([0, 1, 1], [1, 1, 1], 10, 9, 4),          # the same row twice
    ([0, -1, 1], [1, 1, 1], 10, 9, 4), ([0, 4, 1], [1, 1, 1], 10, 9, 4), ([2 ** 31 - 1], [1], 10, 9, 4),
    ([3, 1], [-1, 1], 10, 9, 4), ([3], [-2 ** 31], 10, 9, 4),
    ([0, 0, 9], [40, -1, 1], 2, 0, 15), ([0], [2 ** 31 - 1], 2 ** 20, 0, 11),
])
def test_calls_that_cannot_be_done(dev, seqs, counts, tokens, free, status, inplace):
    """Nothing is changed, and the step has no new tokens."""
    m = Model(1, 4, 8, 4, 30, [3, 4, 0, 9])
    m.stack = m.stack[:free]
    state = m.state(dev)
    before = [t.clone() for t in state]
    s = H.kv_extend(*state, torch.tensor(counts, dtype=I32, device=dev), 4, tokens, inplace=inplace,
                    seqs=torch.tensor(seqs, dtype=I32, device=dev))
    want = m.extend(seqs, counts, tokens)
    assert want[0] == status
    check_step(m, s, seqs, want, False)
    for a, b in zip(before, (state[0], s.lens, state[2], s.n_free)):
        assert torch.equal(a, b)


def test_releases_that_cannot_be_done(dev):
    m = Model(2, 4, 8, 4, 30, [3, 4, 0, 9])
    for seqs, status in (([1, 1], 4), ([-1, 0], 4), ([4], 4)):
        state = m.state(dev)
        r = H.kv_release(*state, 4, seqs=torch.tensor(seqs, dtype=I32, device=dev))
        assert r.status.tolist() == [status]
        check_state(m, state[0], r.lens, state[2], r.n_free)
    # lengths that are not the tables', a stack that would run over
    state = m.state(dev)
    state[1][1] = 2 ** 31 - 1
    r = H.kv_release(*state, 4)
    assert r.status.tolist() == [3] and torch.equal(r.lens, state[1])
    state = m.state(dev)
    state[3][0] = 28
    r = H.kv_release(*state, 4)
    assert r.status.tolist() == [1] and torch.equal(r.lens, state[1]) and r.n_free.tolist() == [28]
    for n, as_if in ((-5, 0), (10 ** 9, 30)):  # such a number of free pages is brought into range
        state = m.state(dev)
        state[3][0] = n
        s = H.kv_extend(*state, torch.zeros(4, dtype=I32, device=dev), 4, 0)
        assert s.status.tolist() == [0] and s.n_free.tolist() == [as_if]


def test_empty_batches(dev):
    m = Model(3, 4, 8, 4, 30, [3, 4, 0, 9])
    state = m.state(dev)
    none = torch.zeros(0, dtype=I32, device=dev)
    s = H.kv_extend(*state, none, 4, 5, seqs=none)
    check_step(m, s, [], m.extend([], [], 5), False)
    r = H.kv_release(*state, 4, seqs=none)
    check_state(m, state[0], r.lens, state[2], r.n_free)
    nobody = Model(4, 0, 8, 4, 30, [])
    s = H.kv_extend(*nobody.state(dev), none, 4, 3)
    assert s.status.tolist() == [0] and s.slots.tolist() == [-1] * 3 and s.n_free.tolist() == [30]
    r = H.kv_release(*nobody.state(dev), 4)
    assert r.status.tolist() == [0] and r.n_free.tolist() == [30]


def test_shared_front_pages_stay(dev):
    """Pages at a row's front that belong to another are not given back."""
    m = Model(5, 3, 8, 4, 30, [17, 9, 8])
    m.tables[1][:2] = m.tables[2][:2] = m.tables[0][:2]
    m.stack = m.stack[:5]
    owned = [0, 2, 2]
    state = m.state(dev)
    o = torch.tensor(owned, dtype=I32, device=dev)
    seqs = torch.tensor([2, 1], dtype=I32, device=dev)
    r = H.kv_release(*state, 4, seqs=seqs, owned_from=o)
    m.release([2, 1], [0, 0], owned)
    check_state(m, state[0], r.lens, state[2], r.n_free)


def test_slots_and_append(dev):
    """kv_append by the slot map writes what kv_append by the tables writes."""
    rng = random.Random(6)
    m = Model(6, 6, 20, 16, 200, [0, 15, 16, 40, 100, 7])
    state = m.state(dev)
    counts = [3, 1, 0, 40, 17, 9]
    s = H.kv_extend(*state, torch.tensor(counts, dtype=I32, device=dev), 16, 80)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((80, 2, 128), generator=g).to(torch.bfloat16).to(dev)[:, ::1] for _ in range(2))
    pools = [torch.zeros((200, 16, 2, 128), dtype=torch.bfloat16, device=dev) for _ in range(4)]
    H.kv_append(k, v, pools[0], pools[1], s.block_table, s.kv_lens, q_starts=s.q_starts)
    H.kv_append(k, v, pools[2], pools[3], slots=s.slots)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3]) and bool(pools[2].any())
    # places outside the pool are skipped, many rows take another path
    big = torch.randn((5000, 2, 128), generator=g).to(torch.bfloat16).to(dev)
    slots = torch.full((5000,), -1, dtype=torch.int64)
    slots[0], slots[1], slots[2], slots[3] = 200 * 16, 2 ** 40, -2 ** 62, 199 * 16 + 15
    slots[4000] = 33
    out = [torch.zeros_like(pools[0]) for _ in range(2)]
    H.kv_append(big, big, out[0], out[1], slots=slots.to(dev))
    want = torch.zeros_like(out[0]).view(3200, 2, 128)
    want[3199], want[33] = big[3], big[4000]
    assert torch.equal(out[0].view(3200, 2, 128), want) and torch.equal(out[1], out[0])


def test_a_decode_loop_in_one_graph(dev):
    """Pages, positions, append and attention of a step captured once: the host takes
    no part in the steps that follow. Two sequences share the first's pages."""
    torch.manual_seed(0)
    page, hk, hq, d, prefix = 16, 2, 8, 64, 48
    rows, width, n_pages = 4, 16, 60
    bf = torch.bfloat16
    k_pages, v_pages = (torch.zeros((n_pages, page, hk, d), dtype=bf, device=dev) for _ in range(2))
    tables = torch.full((rows, width), -1, dtype=I32, device=dev)
    lens = torch.zeros(rows, dtype=I32, device=dev)
    free, n_free = torch.randperm(n_pages, device=dev).to(I32), torch.tensor([n_pages], dtype=I32, device=dev)
    # row 3 holds the prefix, rows 0..2 begin with its pages
    one = torch.tensor([3], dtype=I32, device=dev)
    s = H.kv_extend(tables, lens, free, n_free, torch.tensor([prefix], dtype=I32, device=dev), page, prefix, seqs=one,
                    inplace=True)
    pk, pv = (torch.randn((prefix, hk, d), device=dev).to(bf) for _ in range(2))
    H.kv_append(pk, pv, k_pages, v_pages, slots=s.slots)
    head = tables[3, :prefix // page].clone()
    tables[:3, :prefix // page] = head
    lens[:3] = prefix
    seqs = torch.tensor([2, 0, 1], dtype=I32, device=dev)
    counts = torch.tensor([1, 1, 1], dtype=I32, device=dev)
    q, k, v = (torch.zeros((3, h, d), dtype=bf, device=dev) for h in (hq, hk, hk))

    def step():
        s = H.kv_extend(tables, lens, free, n_free, counts, page, 3, seqs=seqs, inplace=True)
        at = s.positions
        qr = H.rope(q[:, :, None, :], d, base=1e4, offsets=at)[:, :, 0]
        kr = H.rope(k[:, :, None, :], d, base=1e4, offsets=at)[:, :, 0]
        H.kv_append(kr, v, k_pages, v_pages, slots=s.slots)
        o = H.shared_prefix_attention(qr, k_pages, v_pages, s.block_table, s.kv_lens, head, prefix)
        return o, s, qr

    graph = torch.cuda.CUDAGraph()
    saved = [t.clone() for t in (tables, lens, free, n_free, k_pages, v_pages)]
    step()
    for t, u in zip((tables, lens, free, n_free, k_pages, v_pages), saved):
        t.copy_(u)
    with torch.cuda.graph(graph):
        o, s, qr = step()
    for t, u in zip((tables, lens, free, n_free, k_pages, v_pages), saved):
        t.copy_(u)
    for n in range(40):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device=dev).to(bf))
        graph.replay()
        torch.cuda.synchronize()
        assert s.status.tolist() == [0] and lens.tolist()[1] == prefix + n + 1
        if n in (0, 5, 17, 39):
            R.check(o.cpu(), R.attend(qr.cpu(), k_pages.cpu(), v_pages.cpu(), tables[seqs.long()].cpu(),
                                      lens[seqs.long()].cpu()), f"step {n}")
    assert int(n_free) == n_pages - 3 - 9
    r = H.kv_release(tables, lens, free, n_free, page, owned_from=torch.tensor([3, 3, 3, 0], dtype=I32, device=dev),
                     inplace=True)
    assert r.status.tolist() == [0] and int(n_free) == n_pages and sorted(free.tolist()) == list(range(n_pages))
