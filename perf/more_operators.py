"""One step of a continuous batch around the layers' own ops: pages given out and
taken back on the GPU with the step's tables and slot maps, the attention of a
batch over a prompt that all of its sequences share, the routing of tokens to
experts and the sum of the experts' outputs.

Head layouts are those of the workloads in bench.py (Llama-3.2-1B, Qwen3-8B,
Gemma-2-9B and Qwen3-Next layers). Each case runs in elementary torch
operations, or through the framework's public functions where `own` is set.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

F32, F64, I32, I64 = torch.float32, torch.float64, torch.int32, torch.int64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# q heads, kv heads, head_dim
LLAMA, QWEN3, GEMMA, NEXT = (32, 8, 64), (32, 8, 128), (16, 8, 256), (16, 2, 256)

# The largest amount of arithmetic and of traffic that a drawn case has, and the
# scores and cached values that the plain form holds at once for it.
MAX_FLOPS, MAX_BYTES = 290e9, 1000 << 20
MAX_SCORES, MAX_CACHED = 700e6, 1200e6


def _attn(layout, **kw):
    h, hk, d = layout
    case = {"kind": "shared", "heads": h, "kv_heads": hk, "head_dim": d, "page": 16, "dtype": "bf16",
            "window": 0, "sinks": 0, "softcap": 0.0, "q": 1}
    return {**case, **kw}


def listed():
    return [
        # two answers begun from one short system prompt: all latency
        _attn(LLAMA, name="shared_2x300", batch=2, prefix=300, own=5),
        # the continuous batch of bench.py's decode workload behind one long system prompt
        _attn(NEXT, name="shared_64x8192", batch=64, prefix=8192, own=1500, page=32),
        # many samples of one document's summary, the document's end inside a page
        _attn(QWEN3, name="shared_256x4001", batch=256, prefix=4001, own=200, page=64),
        # ragged questions of some tokens each about one long document
        _attn(QWEN3, name="shared_turns_32x16384", batch=32, prefix=16384, own=100, q=33, dtype="f16"),
        # a decode step of 64 sequences out of 96 resident ones, tables of up to 32768 tokens
        {"kind": "extend", "name": "extend_64", "resident": 96, "batch": 64, "kv": 32000, "q": 1,
         "page": 32, "width": 1024},
        # ... and of a batch that is all short chats, with questions of up to 64 tokens
        {"kind": "extend", "name": "extend_1000_ragged", "resident": 1000, "batch": 1000, "kv": 3000,
         "q": 64, "page": 16, "width": 256},
        # the ends of 8 requests out of 64
        {"kind": "release", "name": "release_8", "resident": 64, "batch": 8, "kv": 32000, "page": 32,
         "width": 1024, "keep": False},
        # 512 sequences each give up some drafted tokens that were not accepted
        {"kind": "release", "name": "release_512_drafts", "resident": 512, "batch": 512, "kv": 8000,
         "page": 16, "width": 512, "keep": True},
        # one decode step's routing: 512 experts, top 10 renormalised (bench.py's decode experts)
        {"kind": "route", "name": "route_64", "tokens": 64, "experts": 512, "top_k": 10,
         "scores": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_top": 1,
         "renormalize": True, "scale": 1.0, "dtype": "bf16"},
        # a long prefill's: sigmoid scores, a bias for balance, 4 of 8 groups, top 8
        {"kind": "route", "name": "route_16384_groups", "tokens": 16384, "experts": 256, "top_k": 8,
         "scores": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "group_top": 2,
         "renormalize": True, "scale": 2.5, "dtype": "f32"},
        # the experts' outputs of one decode step, with the gated shared expert
        {"kind": "combine", "name": "combine_64", "tokens": 64, "top_k": 10, "hidden": 2048,
         "shared": True, "dtype": "bf16"},
        # ... and of bench.py's 4096-token prefill
        {"kind": "combine", "name": "combine_4096", "tokens": 4096, "top_k": 10, "hidden": 2048,
         "shared": True, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "extend", "release", "route", "route", "combine"])
    while True:
        c = _draw(rng, kind)
        if kind == "shared":
            keys = c["prefix"] + c["own"] + c["q"]
            if (c["batch"] * c["q"] * c["heads"] * keys > MAX_SCORES
                    or c["batch"] * keys * c["kv_heads"] * c["head_dim"] > MAX_CACHED):
                continue
        w = work(c)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return c


def _draw(rng, kind):
    if kind == "shared":
        layout = rng.choice([LLAMA, QWEN3, GEMMA, NEXT, (12, 12, 64), (32, 32, 96), (28, 4, 128)])
        window = rng.choice([0, 0, 0, _log_int(rng, 64, 16384)])
        return _attn(layout, batch=_log_int(rng, 2, 256), prefix=_log_int(rng, 100, 32768),
                     own=_log_int(rng, 1, 2000), q=rng.choice([1, 1, _log_int(rng, 2, 64)]),
                     page=rng.choice([16, 16, 32, 64, 128, 256]), dtype=rng.choice(["bf16", "bf16", "f16"]),
                     window=window, sinks=rng.choice([0, 4, 64]) if window else 0,
                     softcap=rng.choice([0.0, 0.0, 50.0]))
    if kind in ("extend", "release"):
        page = rng.choice([16, 32, 64])
        resident, kv, q = _log_int(rng, 1, 1000), _log_int(rng, 1, 32000), 0
        batch = rng.choice([resident, rng.randint(1, resident)])
        c = {"kind": kind, "resident": resident, "batch": batch, "kv": kv, "page": page}
        if kind == "extend":
            c["q"] = q = rng.choice([1, _log_int(rng, 1, 2048)])
            while c["batch"] * q > 65536:
                c["batch"] = (c["batch"] + 1) // 2
        else:
            c["keep"] = rng.random() < 0.5
        c["width"] = -(-(kv + q) // page) + rng.randint(0, 8)
        return c
    if kind == "route":
        experts = rng.choice([8, 60, 64, 128, 160, 256, 512])
        grouped = experts % 8 == 0 and experts >= 64 and rng.random() < 0.4
        return {"kind": kind, "tokens": _log_int(rng, 1, 16384), "experts": experts,
                "top_k": rng.randint(1, min(10, experts)), "scores": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": 8 if grouped else 1,
                "top_groups": rng.randint(2, 4) if grouped else 1,
                "group_top": rng.choice([1, 2]) if grouped else 1, "renormalize": rng.random() < 0.6,
                "scale": rng.choice([1.0, 2.5]), "dtype": rng.choice(["bf16", "f16", "f32"])}
    return {"kind": kind, "tokens": _log_int(rng, 1, 4096), "top_k": rng.randint(1, 10),
            "hidden": rng.choice([2048, 2880, 3584, 4096, 7168]), "shared": rng.random() < 0.5,
            "dtype": rng.choice(["bf16", "bf16", "f16"])}


# ------------------------------------------------------------------ sizes
def _rng(case):
    return random.Random("%d %d %d" % (case["batch"], case.get("prefix", case.get("kv", 0)),
                                       case.get("q", 1)))


def _lens(case):
    """(new tokens, tokens with them) of each sequence of an attention case."""
    rng, out = _rng(case), []
    for i in range(case["batch"]):
        q = case["q"] if i == 0 else rng.randint(1, case["q"])
        out.append((q, case["prefix"] + (case["own"] if i == 0 else rng.randint(0, case["own"])) + q))
    return out


def _residents(case):
    """Tokens of each resident sequence; those of the batch with their new tokens, or
    the tokens that they keep."""
    rng = _rng(case)
    lens = [case["kv"] if i == 0 else rng.randint(0, case["kv"]) for i in range(case["resident"])]
    seqs = list(range(case["resident"]))
    if case["batch"] < case["resident"]:
        rng.shuffle(seqs)
        seqs = seqs[:case["batch"]]
    if case["kind"] == "extend":
        # one token each, or ragged turns, some sequences idle
        return lens, seqs, [1 if case["q"] == 1 else rng.randint(0, case["q"]) for _ in seqs]
    return lens, seqs, [max(0, lens[s] - rng.randint(0, 8)) if case["keep"] else 0 for s in seqs]


def work(case):
    kind = case["kind"]
    if kind == "shared":
        d, hk, w, sinks, prefix = (case[k] for k in ("head_dim", "kv_heads", "window", "sinks", "prefix"))
        pairs, keys, tokens, pages, far = 0, 0, 0, 0, prefix
        for q, kv in _lens(case):
            tokens += q
            pages += -(-kv // case["page"])
            first = 0
            for p in range(kv - q, kv):
                lo = max(0, p - w + 1) if w else 0
                pairs += p + 1 - lo + min(sinks, lo)
            if w:
                first = max(0, kv - q - w + 1)
            far = min(far, first)
            # its own keys that one of its queries sees
            lo = max(first, prefix)
            keys += kv - lo + max(0, min(sinks, lo) - prefix)
        keys += prefix - far + min(sinks, far)
        return {"bytes": 2 * keys * hk * d * 2 + 2 * tokens * case["heads"] * d * 2 + 4 * pages,
                "flops": 4 * case["heads"] * d * pairs}
    if kind in ("extend", "release"):
        lens, seqs, n = _residents(case)
        page, moved = case["page"], 0
        for s, m in zip(seqs, n):
            a, b = (lens[s], lens[s] + m) if kind == "extend" else (m, lens[s])
            moved += -(-b // page) - -(-a // page)
        # pages read and written; lengths in and out, counts and sequences
        small = 4 * (2 * len(lens) + 2 * len(seqs) + 4)
        if kind == "release":
            return {"bytes": 8 * moved + small, "flops": 0}
        total = 8 * moved + small + 8 * len(seqs) + 12 * sum(n)
        if case["batch"] < case["resident"]:  # the batch's table, of the rows in its order
            total += sum(4 * -(-(lens[s] + m) // page) for s, m in zip(seqs, n)) + 4 * len(seqs) * case["width"]
        return {"bytes": total, "flops": 0}
    t, k = case["tokens"], case["top_k"]
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "route":
        return {"bytes": t * case["experts"] * size + 8 * t * k + 4 * case["experts"] * case["bias"],
                "flops": 4 * t * case["experts"]}
    rows = t * k + t + (t if case["shared"] else 0)
    return {"bytes": rows * case["hidden"] * size + 4 * t * k + 4 * t * case["shared"],
            "flops": 2 * t * (k + case["shared"]) * case["hidden"]}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*shape, dtype=DTYPES[case.get("dtype", "f32")], std=1.0):
        return torch.empty(shape, dtype=F32, device=dev).normal_(0.0, std, generator=g).to(dtype)

    def perm(n):
        return torch.randperm(n, device=dev, generator=g).to(I32)

    def ints(values):
        return torch.tensor(values, dtype=I32, device=dev)

    st, kind = {"case": case}, case["kind"]
    if kind == "shared":
        d, hk, page, prefix = (case[k] for k in ("head_dim", "kv_heads", "page", "prefix"))
        lens = _lens(case)
        # the prefix's pages, the last of them perhaps not full: its tokens are in the
        # sequences' own pages too, as in a cache whose forks have been written to
        head = -(-prefix // page)
        whole = prefix // page
        need = [-(-kv // page) - whole for _, kv in lens]
        n = head + sum(need) + 3
        order = perm(n)
        st["prefix_table"] = order[:head].clone()
        table = torch.full((len(lens), whole + max(need)), -1, dtype=I32, device=dev)
        table[:, :whole] = order[:whole]
        at = head
        for i, c in enumerate(need):
            table[i, whole:whole + c] = order[at:at + c]
            at += c
        for name in ("k_pages", "v_pages"):
            st[name] = torch.empty((n, page, hk, d), dtype=DTYPES[case["dtype"]], device=dev).normal_(generator=g)
            if head > whole:
                st[name][table[:, whole].long(), :prefix - whole * page] = \
                    st[name][order[whole].long(), :prefix - whole * page]
        starts = [0]
        for q, _ in lens:
            starts.append(starts[-1] + q)
        st["block_table"], st["kv_lens"] = table, ints([kv for _, kv in lens])
        st["q_starts"] = None if case["q"] == 1 else ints(starts)
        st["q_max"], st["kv_max"] = max(q for q, _ in lens), max(kv for _, kv in lens)
        st["q"] = randn(starts[-1], case["heads"], d)
    elif kind in ("extend", "release"):
        lens, seqs, counts = _residents(case)
        page, width = case["page"], case["width"]
        have = [-(-n // page) for n in lens]
        spare = sum(-(-(lens[s] + c) // page) - have[s] for s, c in zip(seqs, counts)) if kind == "extend" else 0
        n_pages = sum(have) + spare + 100
        order = perm(n_pages)
        st["tables"] = torch.full((case["resident"], width), -1, dtype=I32, device=dev)
        at = 0
        for i, c in enumerate(have):
            st["tables"][i, :c] = order[at:at + c]
            at += c
        st["free_pages"] = torch.zeros(n_pages, dtype=I32, device=dev)
        st["free_pages"][:n_pages - at] = order[at:]
        st["n_free"], st["lens"] = ints([n_pages - at]), ints(lens)
        st["seqs"] = ints(seqs) if case["batch"] < case["resident"] else None
        st["counts"] = ints(counts)
        st["keep"] = st["counts"] if kind == "release" and case["keep"] else None
        st["tokens"] = sum(counts) if case.get("q", 1) == 1 else (sum(counts) + 255) // 256 * 256
    elif kind == "route":
        st["logits"] = randn(case["tokens"], case["experts"], std=1.5)
        st["bias"] = randn(case["experts"], dtype=F32, std=0.05) if case["bias"] else None
    else:
        t, k, h = case["tokens"], case["top_k"], case["hidden"]
        st["y"] = randn(t * k, h)
        w = torch.rand((t, k), dtype=F32, device=dev, generator=g)
        st["weights"] = w / w.sum(-1, keepdim=True)
        st["shared"] = randn(t, h) if case["shared"] else None
        st["shared_gate"] = randn(t, 1) if case["shared"] else None
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"shared": _shared, "extend": _extend, "release": _release, "route": _route,
                "combine": _combine}[kind](state)
    import higgs_amd as H

    if kind == "shared":
        return H.shared_prefix_attention(state["q"], state["k_pages"], state["v_pages"], state["block_table"],
                                         state["kv_lens"], state["prefix_table"], case["prefix"],
                                         window=case["window"], sinks=case["sinks"], softcap=case["softcap"],
                                         q_starts=state["q_starts"])
    if kind == "extend":
        s = H.kv_extend(state["tables"], state["lens"], state["free_pages"], state["n_free"], state["counts"],
                        case["page"], state["tokens"], seqs=state["seqs"])
        return (s.block_table, s.kv_lens, s.q_starts, s.slots, s.positions, s.lens, s.n_free, s.status,
                state["tables"])
    if kind == "release":
        s = H.kv_release(state["tables"], state["lens"], state["free_pages"], state["n_free"], case["page"],
                         seqs=state["seqs"], keep=state["keep"])
        return s.lens, s.n_free, s.status, state["free_pages"]
    if kind == "route":
        return H.moe_route(state["logits"], case["top_k"], scores=case["scores"], bias=state["bias"],
                           groups=case["groups"], top_groups=case["top_groups"], group_top=case["group_top"],
                           renormalize=case["renormalize"], scale=case["scale"])
    return H.moe_combine(state["y"], state["weights"], shared=state["shared"], shared_gate=state["shared_gate"])


def _shared(st):
    """Every sequence's attention over its own table, as without sharing."""
    case, q = st["case"], st["q"]
    k_pages, v_pages, lens = st["k_pages"], st["v_pages"], st["kv_lens"].long()
    _, page, hk, d = k_pages.shape
    T, hq, _ = q.shape
    B, Q, L = lens.numel(), st["q_max"], st["kv_max"]
    dev = q.device
    starts = torch.arange(B + 1, device=dev) if st["q_starts"] is None else st["q_starts"].long()
    j = torch.arange(L, device=dev)
    rows = st["block_table"].long()[:, j // page].clamp(min=0) * page + j % page  # [B, L]
    k = k_pages.reshape(-1, hk, d)[rows].to(F32)  # [B, L, Hk, D]
    v = v_pages.reshape(-1, hk, d)[rows].to(F32)
    i = torch.arange(Q, device=dev)
    qi = (starts[:-1, None] + i).clamp(max=T - 1)  # [B, Q]
    qf = q[qi].to(F32).reshape(B, Q, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    s = torch.matmul(qf.reshape(B, hk, -1, d), k.permute(0, 2, 3, 1).contiguous()) * (1.0 / math.sqrt(d))
    s = s.reshape(B, hk, hq // hk, Q, L)
    if case["softcap"]:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    p = (lens - (starts[1:] - starts[:-1]))[:, None] + i  # position of each query [B, Q]
    seen = j <= p[:, :, None]
    if case["window"]:
        seen = seen & ((j > p[:, :, None] - case["window"]) | (j < case["sinks"]))
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    e = torch.exp(s - s.amax(-1, keepdim=True))
    e = e / e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(B, hk, -1, L), v.permute(0, 2, 1, 3).contiguous())
    o = o.reshape(B, hk, hq // hk, Q, d).permute(0, 3, 1, 2, 4).reshape(B, Q, hq, d)
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(starts, t, right=True) - 1
    return o[b, t - starts[b]].to(q.dtype)


def _extend(st):
    tables, lens, free, counts, T = st["tables"], st["lens"], st["free_pages"], st["counts"].long(), st["tokens"]
    page, dev = st["case"]["page"], tables.device
    S, W = tables.shape
    seqs = torch.arange(S, device=dev) if st["seqs"] is None else st["seqs"].long()
    old = lens[seqs].long()
    had, has = (old + page - 1) // page, (old + counts + page - 1) // page
    ends = torch.cumsum(has - had, 0)
    # 1: too few free pages, 2: a sequence outgrows its table, 4: a sequence outside the
    # tables or named twice or a count below zero, 8: more tokens than rows; then nothing is done
    twice = torch.zeros(S, dtype=I64, device=dev).scatter_add_(0, seqs, torch.ones_like(seqs))[seqs] > 1
    status = ((ends[-1] > st["n_free"][0]).long() + 2 * (has > W).any() + 4 * (twice | (counts < 0)).any()
              + 8 * (counts.sum() > T))
    go = status == 0
    counts, has, ends = counts * go, torch.where(go, has, had), ends * go
    j = torch.arange(W, device=dev)
    at = st["n_free"].long() - 1 - ((ends - (has - had))[:, None] + j - had[:, None])
    new = (j >= had[:, None]) & (j < has[:, None])
    rows = torch.where(new, free[at.clamp(0, free.numel() - 1)], tables[seqs])
    tables[seqs] = rows
    out = tables if st["seqs"] is None else torch.where(j < has[:, None], rows, -1)
    kv_lens = (old + counts).to(I32)
    starts = torch.zeros(counts.numel() + 1, dtype=I64, device=dev)
    starts[1:] = torch.cumsum(counts, 0)
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(starts, t, right=True).clamp(max=counts.numel()) - 1
    pos = old[b] + t - starts[b]
    real = t < starts[-1]
    pos = torch.where(real, pos, 0)
    slots = torch.where(real, rows[b, pos // page].long() * page + pos % page, -1)
    new_lens = lens.clone()
    new_lens[seqs] = kv_lens
    return (out, kv_lens, starts.to(I32), slots, pos.to(I32), new_lens,
            (st["n_free"] - ends[-1]).to(I32), status.reshape(1).to(I32), tables)


def _release(st):
    tables, lens, free = st["tables"], st["lens"], st["free_pages"]
    page, dev = st["case"]["page"], tables.device
    S, W = tables.shape
    seqs = torch.arange(S, device=dev) if st["seqs"] is None else st["seqs"].long()
    old = lens[seqs].long()
    keep = torch.zeros_like(old) if st["keep"] is None else torch.minimum(st["keep"].long().clamp(min=0), old)
    had, has = (old + page - 1) // page, (keep + page - 1) // page
    ends = torch.cumsum(had - has, 0)
    twice = torch.zeros(S, dtype=I64, device=dev).scatter_add_(0, seqs, torch.ones_like(seqs))[seqs] > 1
    status = (st["n_free"][0] + ends[-1] > free.numel()).long() + 4 * twice.any()
    go = status == 0
    keep, has, ends = torch.where(go, keep, old), torch.where(go, has, had), ends * go
    j = torch.arange(W, device=dev)
    at = st["n_free"].long() + (ends - (had - has))[:, None] + j - has[:, None]
    given = (j >= has[:, None]) & (j < had[:, None])
    # entries that are not given up go to a place behind the stack
    longer = torch.cat([free, free[:1]])
    longer[torch.where(given, at, free.numel())] = tables[seqs]
    free.copy_(longer[:-1])
    new_lens = lens.clone()
    new_lens[seqs] = keep.to(I32)
    return new_lens, (st["n_free"] + ends[-1]).to(I32), status.reshape(1).to(I32), free


def _route(st):
    """Scores in 64 bits, where two experts' may lie next to each other; equal ones
    go to the lower index."""
    case, x = st["case"], st["logits"].to(F64)
    T, E, G = x.shape[0], x.shape[1], case["groups"]
    if case["scores"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    choice = score if st["bias"] is None else score + st["bias"].to(F64)
    if case["top_groups"] < G:
        best = torch.sort(choice.reshape(T, G, E // G), dim=-1, descending=True).values[..., :case["group_top"]]
        order = torch.sort(best.sum(-1), dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros((T, G), dtype=torch.bool, device=x.device).scatter_(1, order, True)
        choice = choice.masked_fill(~kept.repeat_interleave(E // G, dim=1), float("-inf"))
    experts = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
    w = score.gather(1, experts)
    if case["renormalize"]:
        w = w / w.sum(-1, keepdim=True)
    return (w * case["scale"]).to(F32), experts.to(I32)


def _combine(st):
    w, y = st["weights"], st["y"]
    T, k = w.shape
    rows = torch.where(w[..., None] == 0, 0.0, w[..., None] * y.to(F32).reshape(T, k, -1))
    out = rows.sum(1)
    if st["shared"] is not None:
        out = out + st["shared"].to(F32) / (1.0 + torch.exp(-st["shared_gate"].to(F32)))
    return out.to(y.dtype)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"shared": _exact_shared, "extend": _exact_extend, "release": _exact_release,
            "route": _exact_route, "combine": _exact_combine}[case["kind"]](case, st)


def _exact_shared(case, st):
    page, d, hk = case["page"], case["head_dim"], case["kv_heads"]
    group, at = case["heads"] // hk, 0
    out = torch.empty(st["q"].shape, dtype=F64, device=st["q"].device)
    for b, (nq, kv) in enumerate(_lens(case)):
        pages = st["block_table"][b, :-(-kv // page)].long()
        k, v = (st[n].index_select(0, pages).reshape(-1, hk, d)[:kv].to(F64) for n in ("k_pages", "v_pages"))
        pos = torch.arange(kv - nq, kv, device=k.device).repeat_interleave(group)[:, None]
        key = torch.arange(kv, device=k.device)[None, :]
        hidden = key > pos
        if case["window"]:
            hidden |= (key <= pos - case["window"]) & (key >= case["sinks"])
        q = st["q"][at:at + nq].to(F64) / math.sqrt(d)
        for h in range(hk):
            heads = slice(h * group, (h + 1) * group)
            s = q[:, heads].reshape(-1, d) @ k[:, h].T
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            s[hidden] = -math.inf
            out[at:at + nq, heads] = (torch.softmax(s, dim=-1) @ v[:, h]).reshape(nq, group, d)
        at += nq
    return out


def _exact_extend(case, st):
    lens, seqs, counts = _residents(case)
    tables, page, dev = st["tables"].cpu().numpy(), case["page"], st["tables"].device
    stack = st["free_pages"].cpu().tolist()[:int(st["n_free"])]
    starts, slots, positions = [0], [], []
    for s, c in zip(seqs, counts):
        for p in range(lens[s], lens[s] + c):
            if p % page == 0:
                tables[s, p // page] = stack.pop()
            positions.append(p)
            slots.append(int(tables[s, p // page]) * page + p % page)
        lens[s] += c
        starts.append(starts[-1] + c)
    pad = st["tokens"] - len(slots)
    table = tables
    if st["seqs"] is not None:
        table = np.full((len(seqs), case["width"]), -1, np.int32)
        for i, s in enumerate(seqs):
            n = -(-lens[s] // page)
            table[i, :n] = tables[s, :n]

    def ints(v, dtype=I32):
        return torch.as_tensor(np.asarray(v), device=dev).to(dtype)

    return (ints(table), ints([lens[s] for s in seqs]), ints(starts), ints(slots + [-1] * pad, I64),
            ints(positions + [0] * pad), ints(lens), ints([len(stack)]), ints([0]), ints(tables))


def _exact_release(case, st):
    lens, seqs, keep = _residents(case)
    tables, page, dev = st["tables"].cpu().numpy(), case["page"], st["tables"].device
    free, n = st["free_pages"].cpu().numpy(), int(st["n_free"])
    for s, m in zip(seqs, keep):
        for e in range(-(-m // page), -(-lens[s] // page)):
            free[n] = tables[s, e]
            n += 1
        lens[s] = m
    return tuple(torch.as_tensor(np.asarray(v, np.int32), device=dev) for v in (lens, [n], [0], free))


def _exact_route(case, st):
    x = st["logits"].to(F64).cpu().numpy()
    T, E = x.shape
    if case["scores"] == "softmax":
        score = np.exp(x - x.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    else:
        score = 1.0 / (1.0 + np.exp(-x))
    choice = score.copy()
    if st["bias"] is not None:
        choice += st["bias"].to(F64).cpu().numpy()
    if case["groups"] > 1:
        parts = np.sort(choice.reshape(T, case["groups"], -1), axis=2)[:, :, -case["group_top"]:].sum(2)
        for g in np.argsort(-parts, axis=1, kind="stable")[:, case["top_groups"]:].T:
            width = E // case["groups"]
            for i in range(width):
                choice[np.arange(T), g * width + i] = -np.inf
    experts = np.argsort(-choice, axis=1, kind="stable")[:, :case["top_k"]]
    w = np.take_along_axis(score, experts, 1)
    if case["renormalize"]:
        w = w / w.sum(1, keepdims=True)
    dev = st["logits"].device
    return torch.as_tensor(w * case["scale"], device=dev), torch.as_tensor(experts.astype(np.int32), device=dev)


def _exact_combine(case, st):
    T, k, h = case["tokens"], case["top_k"], case["hidden"]
    out = torch.zeros((T, h), dtype=F64, device=st["y"].device)
    for i in range(k):
        out += st["weights"][:, i:i + 1].to(F64) * st["y"][i::k].to(F64)
    if case["shared"]:
        out += torch.sigmoid(st["shared_gate"].to(F64)) * st["shared"].to(F64)
    return out
