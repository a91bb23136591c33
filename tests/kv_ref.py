"""The paged attention's definition in 64 bits, with an error bound for every
element that follows from the kernels' roundings.

Counted, for a type with half step u = finfo.eps / 2 and f32 sums (2^-24):
  - a score is an f32 sum of D products, then scaled (and soft-capped), and
    its exponential's argument is rounded once more: absolute error
    ds <= (D + 4) 2^-24 scale sum |q_d k_d| + 2^-21 (|s| + 1) (2^-21: the
    hardware exp2 and the soft cap's tanh are good to a few f32 ulps of
    values up to the score's own size);
  - a probability carries e^ds - 1 of that and is rounded to the type (u);
    the sum that normalises it carries the ds alone;
  - the weighted sum of n values is an f32 sum (n 2^-24) and the result is
    rounded once to the type.
So |error| <= u |o| + sum_j p_j |v_j| (u + 4 max ds + 2 n 2^-24), plus, for
f16, half the subnormal step 2^-24 for each probability (their sum is at
least 1 where they are rounded) and for the result."""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def gather(pages, table_row, n):
    """Tokens 0..n-1 of a sequence [n, Hk, D] in f64, and which of them exist."""
    n_pages, ps, hk, d = pages.shape
    out = torch.zeros((n, hk, d), dtype=F64)
    there = torch.zeros(n, dtype=torch.bool)
    for e in range(-(-n // ps)):
        page = int(table_row[e]) if e < table_row.numel() else -1
        m = min(ps, n - e * ps)
        if 0 <= page < n_pages:
            out[e * ps:e * ps + m] = pages[page, :m].to(F64)
            there[e * ps:e * ps + m] = True
    return out, there


def seen_mask(p, n, window, sinks):
    """Keys 0..n-1 that the query at position p sees."""
    j = torch.arange(n)
    m = j <= p
    if window > 0:
        m &= (j > p - window) | (j < sinks)
    return m


def attend(q, k_pages, v_pages, table, lens, starts=None, *, scale=None, window=0, sinks=0,
           softcap=0.0):
    """(out, bound, owned) in f64 for CPU tensors; rows of no sequence are not
    owned."""
    T, hq, d = q.shape
    hk = k_pages.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros((T, hq, d), dtype=F64)
    bound = torch.zeros_like(out)
    owned = torch.zeros(T, dtype=torch.bool)
    group = hq // hk
    for b in range(lens.numel()):
        first, stop = (b, b + 1) if starts is None else (int(starts[b]), int(starts[b + 1]))
        n, length = stop - first, int(lens[b])
        if n <= 0:
            continue
        owned[first:stop] = True
        k, there = gather(k_pages, table[b], max(0, length))
        v, _ = gather(v_pages, table[b], max(0, length))
        for i in range(n):
            p = length - n + i
            m = seen_mask(p, max(0, length), window, sinks) & there
            if p < 0 or not bool(m.any()):
                continue
            km, vm = k[m], v[m]  # [n, Hk, D]
            qi = q[first + i].to(F64).reshape(hk, group, d)
            s = torch.einsum("hgd,nhd->hgn", qi, km) * scale
            mag = torch.einsum("hgd,nhd->hgn", qi.abs(), km.abs()) * abs(scale)
            if softcap > 0:
                s = softcap * torch.tanh(s / softcap)
            ds = (d + 4) * 2.0 ** -24 * mag + 2.0 ** -21 * (s.abs() + 1)
            w = torch.softmax(s, -1)
            o = torch.einsum("hgn,nhd->hgd", w, vm)
            a = torch.einsum("hgn,nhd->hgd", w, vm.abs())
            nk = km.shape[0]
            e = u * o.abs() + a * (u + 4 * ds.amax(-1, keepdim=True) + 2 * nk * 2.0 ** -24)
            if q.dtype == torch.float16:
                e = e + 2.0 ** -25 * (1 + vm.abs().sum(0)[:, None, :])
            out[first + i] = o.reshape(hq, d)
            bound[first + i] = e.reshape(hq, d)
    return out, bound, owned


def check(got, ref, what=""):
    """got (CPU tensor) against attend()'s result."""
    out, bound, owned = ref
    g = got.to(F64)
    both = owned[:, None, None].expand_as(out)
    assert torch.equal(torch.isnan(g)[both], torch.isnan(out)[both]), f"{what}: NaN places differ"
    fine = both & torch.isfinite(out)
    err = (g - out).abs()
    bad = fine & ~(err <= bound)
    if bool(bad.any()):
        i = tuple(int(x) for x in torch.nonzero(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {int(fine.sum())} elements beyond the bound; "
                             f"first at {i}: got {float(g[i])}, exact {float(out[i])}, bound {float(bound[i])}")


def make(seed, lens, *, heads, kv_heads, head_dim, page, dtype, news=None, spare=3, head_major=False,
         q_scale=1.0):
    """CPU inputs of a call: q, k_pages, v_pages, table, lens, starts. Pages are
    shuffled; every place that holds no token of a sequence is NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [max(0, -(-n // page)) for n in lens]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g)
    table = torch.full((len(lens), max([*need, 1])), -1, dtype=torch.int32)
    shape = (n_pages, kv_heads, page, head_dim) if head_major else (n_pages, page, kv_heads, head_dim)
    pools = []
    for _ in range(2):
        t = torch.full(shape, float("nan"), dtype=dtype)
        pools.append(t.transpose(1, 2) if head_major else t)
    at = 0
    for b, n in enumerate(lens):
        for e in range(need[b]):
            page_id = int(order[at])
            at += 1
            table[b, e] = page_id
            m = min(page, n - e * page)
            for t in pools:
                t[page_id, :m] = torch.randn((m, kv_heads, head_dim), generator=g).to(dtype)
    starts = None
    rows = len(lens)
    if news is not None:
        starts = torch.tensor([0, *torch.tensor(news).cumsum(0).tolist()], dtype=torch.int32)
        rows = int(starts[-1])
    q = (q_scale * torch.randn((rows, heads, head_dim), generator=g)).to(dtype)
    return {"q": q, "k_pages": pools[0], "v_pages": pools[1], "table": table,
            "lens": torch.tensor(lens, dtype=torch.int32), "starts": starts}


def to(inputs, dev):
    """The same on the device, strides kept."""
    out = {}
    for name, t in inputs.items():
        if t is None:
            out[name] = None
            continue
        d = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev)
        out[name] = d.copy_(t)
    return out


def call(H, x, **kw):
    """paged_attention over make()'s inputs on the device."""
    return H.paged_attention(x["q"], x["k_pages"], x["v_pages"], x["table"], x["lens"],
                             q_starts=x["starts"], **kw)


def reference(x, **kw):
    return attend(x["q"], x["k_pages"], x["v_pages"], x["table"], x["lens"], x["starts"], **kw)
