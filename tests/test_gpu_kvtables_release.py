"""kv_release of named sequences on both sides of where it takes two launches."""
from __future__ import annotations

import random

import pytest
import torch

import higgs_amd as H

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [639, 640, 641, 900, 1024, 1025])
@pytest.mark.parametrize("inplace", [False, True])
def test_named_sequences(dev, batch, inplace):
    rng = random.Random(batch)
    rows, page, width = batch + 60, 16, 12
    lens = [rng.randint(0, page * width) for _ in range(rows)]
    order = list(range(rows * width))
    rng.shuffle(order)
    tables = [[order.pop() if e * page < n else -1 for e in range(width)] for n in lens]
    n_pages = rows * width
    stack = order[:50]
    seqs = rng.sample(range(rows), batch)
    keep = [rng.choice([-1, 0, lens[s] // 2, lens[s], lens[s] + 5]) for s in seqs]
    owned = [rng.randint(0, 3) for _ in range(rows)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    t, ln, free, n = i32(tables), i32(lens), i32(stack + [-7] * (n_pages - 50)), i32([50])
    s = H.kv_release(t, ln, free, n, page, seqs=i32(seqs), keep=i32(keep), owned_from=i32(owned), inplace=inplace)
    for q, k in zip(seqs, keep):
        now = min(max(k, 0), lens[q])
        stack += tables[q][max(-(-now // page), owned[q]):-(-lens[q] // page)]
        lens[q] = now
    assert s.status.item() == 0 and s.n_free.item() == len(stack)
    assert s.lens.tolist() == lens and free.tolist() == stack + [-7] * (n_pages - len(stack))
    assert t.tolist() == tables and (s.lens is ln) == inplace
