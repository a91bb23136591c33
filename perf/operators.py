"""The paged key-value cache and the attention that reads it: single tokens and
prompts over pages, the write of new tokens' keys and values, and page copies.

Head layouts are those of the workloads in bench.py (Llama-3.2-1B, Qwen3-8B,
Gemma-2-9B and Qwen3-Next layers). Each case runs in elementary torch
operations, or through the framework's public functions where `own` is set.
"""
from __future__ import annotations

import math
import random

import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}

# q heads, kv heads, head_dim
LLAMA, QWEN3, GEMMA, NEXT = (32, 8, 64), (32, 8, 128), (16, 8, 256), (16, 2, 256)

# The largest amount of arithmetic and of traffic that a drawn case has, and the
# scores and cached values that the plain form holds at once for it.
MAX_FLOPS, MAX_BYTES = 300e9, 2200 << 20
MAX_SCORES, MAX_CACHED = 1200e6, 2200e6


def _attn(kind, layout, **kw):
    h, hk, d = layout
    case = {"kind": kind, "heads": h, "kv_heads": hk, "head_dim": d, "page": 16, "dtype": "bf16",
            "window": 0, "sinks": 0, "softcap": 0.0, "ragged": False}
    return {**case, **kw}


def listed():
    return [
        # one user's next token early in a chat: all latency
        _attn("decode", LLAMA, name="decode_1x127", batch=1, kv=127),
        # one user far into a long document
        _attn("decode", QWEN3, name="decode_1x131071", batch=1, kv=131071, page=64),
        # the continuous batch of bench.py's decode workload: 64 ragged caches up to 32768
        _attn("decode", NEXT, name="decode_64_ragged", batch=64, kv=32768, ragged=True, page=32),
        # a sliding-window layer with soft-capped scores, first tokens kept visible
        _attn("decode", GEMMA, name="decode_16_window", batch=16, kv=8000, window=4096, sinks=4,
              softcap=50.0, dtype="f16"),
        # four prompts of 1024 tokens (bench.py's Llama chain)
        _attn("prompt", LLAMA, name="prompt_4x1024", batch=4, q=1024, prefix=0),
        # eight prompts of 2048 tokens (bench.py's Qwen3-8B prefill)
        _attn("prompt", QWEN3, name="prompt_8x2048", batch=8, q=2048, prefix=0, page=64),
        # a long prompt of odd length through a sliding-window layer with soft-capped scores
        _attn("prompt", GEMMA, name="prompt_8191_window", batch=1, q=8191, prefix=0, window=4096,
              sinks=4, softcap=50.0),
        # ragged turns of a chat over long cached prefixes, window and first tokens visible
        _attn("prompt", QWEN3, name="prompt_turns_window", batch=6, q=300, prefix=20000, ragged=True,
              window=1024, sinks=4, dtype="f16"),
        # the write of one decode step's keys and values
        {"kind": "append", "name": "append_64", "batch": 64, "q": 1, "prefix": 1000, "ragged": True,
         "kv_heads": 2, "head_dim": 256, "page": 32, "dtype": "bf16"},
        # ... and of eight prompts
        {"kind": "append", "name": "append_8x2048", "batch": 8, "q": 2048, "prefix": 0,
         "ragged": False, "kv_heads": 8, "head_dim": 128, "page": 64, "dtype": "bf16"},
        # a forked sequence writes to its shared last page: one page of 16 layers is copied
        {"kind": "copy", "name": "fork_1", "layers": 16, "pages": 200, "moved": 1, "kv_heads": 8,
         "head_dim": 64, "page": 16, "dtype": "bf16"},
        # compaction after long sequences ended: live pages move down, 12 layers at a time
        {"kind": "copy", "name": "compact_80", "layers": 12, "pages": 200, "moved": 80,
         "kv_heads": 2, "head_dim": 256, "page": 32, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "prompt", "append", "copy"])
    while True:
        c = _draw(rng, kind)
        if c["kind"] in ("decode", "prompt"):
            q, kv = c.get("q", 1), c.get("kv", 0) + c.get("q", 0) + c.get("prefix", 0)
            if (c["batch"] * kv * q * c["heads"] > MAX_SCORES
                    or c["batch"] * kv * c["kv_heads"] * c["head_dim"] * 2 > MAX_CACHED):
                continue
        w = work(c)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return c


def _draw(rng, kind):
    layout = rng.choice([LLAMA, QWEN3, GEMMA, NEXT, (12, 12, 64), (32, 32, 96), (28, 4, 128)])
    page, dtype = rng.choice([16, 16, 32, 64, 128, 256]), rng.choice(["bf16", "bf16", "f16"])
    if kind in ("decode", "prompt"):
        opts = {"page": page, "dtype": dtype, "ragged": rng.random() < 0.6,
                "window": rng.choice([0, 0, _log_int(rng, 1, 8192)]),
                "softcap": rng.choice([0.0, 0.0, 50.0])}
        opts["sinks"] = rng.choice([0, 1, 4, 64]) if opts["window"] else 0
        if kind == "decode":
            return _attn(kind, layout, batch=_log_int(rng, 1, 128), kv=_log_int(rng, 1, 131072), **opts)
        return _attn(kind, layout, batch=rng.randint(1, 8), q=_log_int(rng, 1, 8192),
                     prefix=rng.choice([0, _log_int(rng, 1, 32768)]), **opts)
    if kind == "append":
        return {"kind": kind, "batch": rng.randint(1, 64), "q": rng.choice([1, _log_int(rng, 1, 1024)]),
                "prefix": _log_int(rng, 1, 1024), "ragged": rng.random() < 0.6,
                "kv_heads": layout[1], "head_dim": layout[2], "page": page, "dtype": dtype}
    pages = rng.randint(8, 200)
    return {"kind": kind, "layers": rng.randint(1, 16), "pages": pages,
            "moved": _log_int(rng, 1, pages // 2), "kv_heads": layout[1] // 2, "head_dim": layout[2],
            "page": rng.choice([16, 32]), "dtype": dtype}


# ------------------------------------------------------------------ sizes
def _lens(case):
    """(new tokens, cached tokens including them) of each sequence."""
    rng = random.Random("%d %d" % (case["batch"], case.get("kv", 0) + case.get("q", 0)))

    def some(n, i):
        return n if i == 0 or not case["ragged"] else rng.randint(min(1, n), n)

    if case["kind"] == "decode":
        return [(1, some(case["kv"], i)) for i in range(case["batch"])]
    out = []
    for i in range(case["batch"]):
        q, prefix = some(case["q"], i), some(case["prefix"], i)
        out.append((q, q + prefix))
    return out


def _seen(case, q, kv):
    """(query, key) pairs of one sequence that the mask leaves, and the keys that any query sees."""
    w, s = case["window"], case["sinks"]
    p0 = kv - q
    if not w:
        return q * p0 + q * (q + 1) // 2, kv
    pairs = 0
    for p in range(p0, kv):
        lo = max(0, p - w + 1)
        pairs += p + 1 - lo + min(s, lo)
    lo = max(0, p0 - w + 1)
    return pairs, kv - lo + min(s, lo)


def work(case):
    d, hk = case["head_dim"], case["kv_heads"]
    if case["kind"] == "copy":
        moved = case["moved"] * case["layers"] * case["page"] * hk * d * 2 * 2
        return {"bytes": 2 * moved + 8 * case["moved"], "flops": 0}
    lens = _lens(case)
    pages = sum(-(-kv // case["page"]) for _, kv in lens)
    tokens = sum(q for q, _ in lens)
    if case["kind"] == "append":
        return {"bytes": 2 * 2 * tokens * hk * d * 2 + 4 * (pages + 2 * len(lens)), "flops": 0}
    pairs = keys = 0
    for q, kv in lens:
        n, k = _seen(case, q, kv)
        pairs += n
        keys += k
    return {"bytes": 2 * keys * hk * d * 2 + 2 * tokens * case["heads"] * d * 2 + 4 * (pages + 2 * len(lens)),
            "flops": 4 * case["heads"] * d * pairs}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev, dt = torch.device("cuda", torch.cuda.current_device()), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.empty(shape, dtype=dt, device=dev).normal_(generator=g)

    d, hk, page = case["head_dim"], case["kv_heads"], case["page"]
    st = {"case": case}
    if case["kind"] == "copy":
        n, m = case["pages"], case["moved"]
        st["k_pages"], st["v_pages"] = (randn(case["layers"], n, page, hk, d) for _ in range(2))
        # which pages move where is known on the host, where pages are given out
        perm = torch.randperm(n, device=dev, generator=g).tolist()
        st["src"], st["dst"] = perm[:m], perm[m:2 * m]
        return st
    lens = _lens(case)
    need = [-(-kv // page) for _, kv in lens]
    n = sum(need) + 3
    st["k_pages"], st["v_pages"] = (randn(n, page, hk, d) for _ in range(2))
    perm = torch.randperm(n, device=dev, generator=g).to(torch.int32)
    table = torch.zeros((len(lens), max(need)), dtype=torch.int32, device=dev)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = perm[at:at + c]
        at += c
    starts = [0]
    for q, _ in lens:
        starts.append(starts[-1] + q)
    st["block_table"] = table
    st["kv_lens"] = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=dev)
    # one token a sequence needs no starts
    st["q_starts"] = (None if case["kind"] == "decode" or case["kind"] == "append" and case["q"] == 1
                      else torch.tensor(starts, dtype=torch.int32, device=dev))
    st["q_max"], st["kv_max"] = max(q for q, _ in lens), max(kv for _, kv in lens)
    if case["kind"] == "append":
        st["k"], st["v"] = randn(starts[-1], hk, d), randn(starts[-1], hk, d)
    else:
        st["q"] = randn(starts[-1], case["heads"], d)
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        import higgs_amd as H

        if case["kind"] == "copy":
            H.kv_copy_pages(state["k_pages"], state["v_pages"], state["src"], state["dst"])
            return state["k_pages"], state["v_pages"]
        at = (state["k_pages"], state["v_pages"], state["block_table"], state["kv_lens"])
        if case["kind"] == "append":
            H.kv_append(state["k"], state["v"], *at, q_starts=state["q_starts"])
            return state["k_pages"], state["v_pages"]
        return H.paged_attention(state["q"], *at, window=case["window"], sinks=case["sinks"],
                                 softcap=case["softcap"], q_starts=state["q_starts"])
    return {"copy": _copy, "append": _append, "decode": _attend, "prompt": _attend}[case["kind"]](state)


def _copy(st):
    k, v = st["k_pages"], st["v_pages"]
    src, dst = torch.tensor(st["src"], device=k.device), torch.tensor(st["dst"], device=k.device)
    k[:, dst] = k[:, src]
    v[:, dst] = v[:, src]
    return k, v


def _starts(st):
    if st["q_starts"] is not None:
        return st["q_starts"].long()
    return torch.arange(st["kv_lens"].numel() + 1, device=st["kv_lens"].device)


def _of_token(st, tokens):
    """The sequence of each token, and its place among the sequence's new tokens."""
    starts = _starts(st)
    t = torch.arange(tokens, device=starts.device)
    b = torch.searchsorted(starts, t, right=True) - 1
    return b, t - starts[b]


def _append(st):
    k, page = st["k"], st["k_pages"].shape[1]
    b, i = _of_token(st, k.shape[0])
    starts, lens = _starts(st), st["kv_lens"].long()
    at = lens[b] - (starts[b + 1] - starts[b]) + i
    rows = st["block_table"].long()[b, at // page]
    st["k_pages"][rows, at % page] = k
    st["v_pages"][rows, at % page] = st["v"]
    return st["k_pages"], st["v_pages"]


def _attend(st):
    case, q = st["case"], st["q"]
    k_pages, v_pages, lens = st["k_pages"], st["v_pages"], st["kv_lens"].long()
    _, page, hk, d = k_pages.shape
    T, hq, _ = q.shape
    B, Q, L = lens.numel(), st["q_max"], st["kv_max"]
    j = torch.arange(L, device=q.device)
    rows = st["block_table"].long()[:, j // page] * page + j % page  # [B, L]
    k = k_pages.reshape(-1, hk, d)[rows].to(F32)  # [B, L, Hk, D]
    v = v_pages.reshape(-1, hk, d)[rows].to(F32)
    starts = _starts(st)
    i = torch.arange(Q, device=q.device)
    qi = (starts[:-1, None] + i).clamp(max=T - 1)  # [B, Q]
    qf = q[qi].to(F32).reshape(B, Q, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    s = torch.matmul(qf.reshape(B, hk, -1, d), k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
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
    o = torch.matmul(e.reshape(B, hk, -1, L), v.permute(0, 2, 1, 3))
    o = o.reshape(B, hk, hq // hk, Q, d).permute(0, 3, 1, 2, 4).reshape(B, Q, hq, d)
    b, at = _of_token(st, T)
    return o[b, at].to(q.dtype)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "copy":
        out = []
        for name in ("k_pages", "v_pages"):
            old = st[name].to(F64)
            new = old.clone()
            for s, t in zip(st["src"], st["dst"]):
                new[:, t] = old[:, s]
            out.append(new)
        return tuple(out)
    page, lens, table = case["page"], _lens(case), st["block_table"].tolist()
    if case["kind"] == "append":
        out = []
        for name in ("k", "v"):
            pool, new, at = st[name + "_pages"].to(F64), st[name].to(F64), 0
            for b, (q, kv) in enumerate(lens):
                first = kv - q
                while first < kv:
                    stop = min(kv, (first // page + 1) * page)
                    pool[table[b][first // page], first % page:first % page + stop - first] = \
                        new[at:at + stop - first]
                    at += stop - first
                    first = stop
            out.append(pool)
        return tuple(out)
    d, hk, group = case["head_dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    out, at = torch.empty(st["q"].shape, dtype=F64, device=st["q"].device), 0
    for b, (nq, kv) in enumerate(lens):
        pages = st["block_table"][b, :-(-kv // page)].long()
        k, v = (st[n].index_select(0, pages).reshape(-1, hk, d)[:kv].to(F64) for n in ("k_pages", "v_pages"))
        q = st["q"][at:at + nq].to(F64) / math.sqrt(d)
        pos = torch.arange(kv - nq, kv, device=q.device)[:, None]
        key = torch.arange(kv, device=q.device)[None, :]
        hidden = key > pos
        if case["window"]:
            hidden |= (key <= pos - case["window"]) & (key >= case["sinks"])
        for h in range(case["heads"]):
            s = q[:, h] @ k[:, h // group].T
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            s[hidden] = -math.inf
            w = torch.softmax(s, dim=-1)
            out[at:at + nq, h] = w @ v[:, h // group]
        at += nq
    return out
