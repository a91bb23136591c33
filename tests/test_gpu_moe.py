"""moe_route and moe_combine against their definitions in 64 bits.

Counted, with half a step of f32 at 2^-24: a weight's exponentials are good to
2^-22 of themselves (the hardware's exp2 to one step, 2^-23, the rest its
argument's), a sum of n of them adds n 2^-24, a quotient and a product 2^-24 each;
renormalising divides by a sum of such values once more. So a weight is within
(2 * 2^-22 + (n + top_k + 6) 2^-24) of itself. A sum over top_k rows is f32:
(top_k + 3) 2^-24 of the magnitudes added, the gate 2^-21 of its row's, and half a
step of the result's type."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import higgs_amd as H

pytestmark = pytest.mark.gpu

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def route(x, top_k, *, scores="softmax", bias=None, groups=1, top_groups=1, group_top=1, renormalize=False, scale=1.0):
    """(weights, experts) in 64 bits, a token at a time."""
    x = x.to(F64).numpy()
    W, X = [], []
    for l in x:
        l = np.where(np.isnan(l), -np.inf, l)
        E = len(l)
        if scores == "softmax":
            top = l.max()
            e = np.where(l == top, 1.0, np.exp(np.where(np.isfinite(l), l, -np.inf) - (top if np.isfinite(top) else 0.0)))
            if top == np.inf:
                e = (l == np.inf).astype(float)
            if top == -np.inf:
                e = np.zeros(E)
            s = e / e.sum() if e.sum() > 0 else e
            order = l
        else:
            s = 1.0 / (1.0 + np.exp(-l))
            order = l
        if bias is not None or (group_top == 2 and top_groups < groups):
            order = s + (0.0 if bias is None else bias.to(F64).numpy())
        order = np.where(np.isnan(order), -np.inf, order)
        allowed = np.ones(E, bool)
        if top_groups < groups:
            parts = [sum(sorted(order[g * (E // groups):(g + 1) * (E // groups)])[-group_top:]) for g in range(groups)]
            kept = sorted(range(groups), key=lambda g: (-parts[g], g))[:top_groups]
            allowed = np.repeat([g in kept for g in range(groups)], E // groups)
        best = sorted((i for i in range(E) if allowed[i]), key=lambda i: (-order[i], i))[:top_k]
        w = s[best]
        if renormalize:
            w = w / w.sum() if w.sum() > 0 else w
        W.append(w * scale)
        X.append(best)
    return torch.tensor(np.array(W)).reshape(len(x), top_k), torch.tensor(np.array(X), dtype=torch.int32).reshape(len(x), top_k)


def check_route(dev, x, top_k, **kw):
    w, e = H.moe_route(x.to(dev), top_k, **{k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    rw, re = route(x, top_k, **kw)
    assert w.dtype == F32 and e.dtype == torch.int32 and w.shape == e.shape == (x.shape[0], top_k)
    assert torch.equal(e.cpu(), re), (e.cpu() != re).nonzero()[:5]
    bound = rw.abs() * (2 * 2.0 ** -22 + (x.shape[1] + top_k + 6) * 2.0 ** -24) + 1e-37
    err = (w.cpu().to(F64) - rw).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("experts,top_k", [(1, 1), (2, 2), (8, 2), (60, 4), (63, 63), (64, 64), (65, 6), (128, 8), (160, 6),
                                           (256, 8), (257, 33), (512, 10), (1000, 7), (1024, 64)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_sizes(dev, experts, top_k, scores, dtype):
    g = torch.Generator().manual_seed(experts)
    for tokens, renormalize, scale in ((1, False, 1.0), (37, True, 2.5)):
        x = (2 * torch.randn((tokens, experts), generator=g)).to(dtype)
        check_route(dev, x, top_k, scores=scores, renormalize=renormalize, scale=scale)
        bias = 0.2 * torch.randn((experts,), generator=g)
        check_route(dev, x, top_k, scores=scores, renormalize=renormalize, scale=scale, bias=bias)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("experts,groups,top_groups,group_top,top_k", [
    (256, 8, 4, 2, 8), (160, 8, 3, 1, 6), (256, 8, 4, 1, 8), (64, 64, 5, 1, 5), (64, 32, 7, 2, 9), (24, 3, 2, 2, 5),
    (60, 5, 1, 2, 12), (1024, 64, 64, 2, 8), (1024, 64, 3, 2, 40), (512, 2, 1, 2, 64), (512, 16, 1, 1, 32), (6, 6, 6, 1, 6),
    (72, 9, 2, 2, 3)])
def test_route_groups(dev, experts, groups, top_groups, group_top, top_k, bias, scores):
    g = torch.Generator().manual_seed(experts + groups)
    x = (1.5 * torch.randn((50, experts), generator=g)).to(F32)
    b = 0.1 * torch.randn((experts,), generator=g) if bias else None
    check_route(dev, x, top_k, scores=scores, bias=b, groups=groups, top_groups=top_groups, group_top=group_top,
                renormalize=True)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_equal_scores_go_to_the_lower_expert(dev, scores, bias):
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-2, 3, (200, 256), generator=g).to(BF16)
    b = torch.randint(0, 2, (256,), generator=g).to(F32) * 0.25 if bias else None
    check_route(dev, x, 20, scores=scores, bias=b)
    check_route(dev, x, 12, scores=scores, bias=b, groups=8, top_groups=3, group_top=1)
    check_route(dev, torch.zeros((3, 100), dtype=F16), 9, scores=scores)
    check_route(dev, torch.tensor([[0.0, -0.0, -0.0, 0.0] * 20], dtype=BF16), 5, scores=scores)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_masked_and_odd_logits(dev, scores, bias, dtype):
    """-inf, the type's lowest value, +inf and NaN; rows that they leave empty."""
    inf, nan, low = float("inf"), float("nan"), torch.finfo(dtype).min
    g = torch.Generator().manual_seed(4)
    x = torch.randn((9, 70), generator=g).to(dtype)
    x[0] = -inf
    x[1] = nan
    x[2] = low
    x[3, 5:] = -inf
    x[4, 3:] = low
    x[5, 7] = nan
    x[6, [2, 9]] = inf
    x[7, ::2] = -inf
    x[7, 1::4] = nan
    x[8] = -inf
    x[8, 69] = 1.0
    b = 0.1 * torch.randn((70,), generator=g) if bias else None
    for kw in ({}, {"renormalize": True}, {"groups": 10, "top_groups": 2, "group_top": 2, "renormalize": True}):
        check_route(dev, x, 8, scores=scores, bias=b, **kw)
    if bias:  # experts that are switched off, and forced ones
        b[3], b[4], b[5], b[69] = -inf, inf, nan, inf
        check_route(dev, x, 8, scores=scores, bias=b)
        check_route(dev, x, 64, scores=scores, bias=b)


def test_route_close_choices(dev):
    """Sums of a score and a bias that f32 does not tell apart."""
    x = torch.zeros((1, 128), dtype=F32)
    x[0] = torch.arange(128) * 2.0 ** -26
    check_route(dev, x, 10, scores="sigmoid", bias=torch.full((128,), 3.0))
    check_route(dev, x.flip(1), 10, scores="sigmoid", bias=torch.full((128,), 3.0))
    x = torch.linspace(20, 30, 128)[None]
    check_route(dev, x, 10, scores="sigmoid", bias=torch.full((128,), 0.5))


def test_route_layouts(dev):
    g = torch.Generator().manual_seed(5)
    wide = torch.randn((30, 300), generator=g).to(BF16)
    for cols in (slice(0, 128), slice(7, 135), slice(1, 257)):
        d = wide.to(dev)[:, cols]
        w, e = H.moe_route(d, 6, renormalize=True)
        rw, re = route(wide[:, cols], 6, renormalize=True)
        assert torch.equal(e.cpu(), re) and float((w.cpu().to(F64) - rw).abs().max()) < 1e-5
    d = wide.to(dev)[:, :64]
    w, e = H.moe_route(d.reshape(5, 6, 64), 3)
    w2, e2 = H.moe_route(d, 3)
    assert w.shape == (5, 6, 3) and torch.equal(w.reshape(30, 3), w2) and torch.equal(e.reshape(30, 3), e2)
    w1, e1 = H.moe_route(d[4], 3)
    assert torch.equal(w1, w2[4]) and torch.equal(e1, e2[4])
    w0, e0 = H.moe_route(d[:0], 3)
    assert w0.shape == e0.shape == (0, 3)


def test_route_does_not_depend_on_the_batch(dev):
    """A token's experts and weights are the same bits in any batch, every time."""
    g = torch.Generator().manual_seed(6)
    for experts, kw in ((512, dict(renormalize=True)), (256, dict(scores="sigmoid", groups=8, top_groups=4, group_top=2)),
                        (100, dict(bias=torch.randn((100,), generator=g).to(dev)))):
        x = torch.randn((3000, experts), generator=g).to(BF16).to(dev)
        w, e = H.moe_route(x, 8, **kw)
        for a, b in ((0, 1), (17, 30), (1000, 2999)):
            w2, e2 = H.moe_route(x[a:b], 8, **kw)
            assert torch.equal(w[a:b], w2) and torch.equal(e[a:b], e2)


def combine(y, w, shared=None, gate=None):
    """(result, bound) in 64 bits."""
    T, k = w.shape
    rows = y.to(F64).reshape(T, k, -1)
    rows = torch.where(w[..., None] == 0, 0.0, w.to(F64)[..., None] * rows)
    out, mag = rows.sum(1), rows.abs().sum(1)
    bound = (k + 3) * 2.0 ** -24 * mag
    if shared is not None:
        s = shared.to(F64)
        if gate is not None:
            s = s * torch.sigmoid(gate.to(F64)).reshape(T, 1)
        out = out + s
        bound = bound + s.abs() * (2.0 ** -21 + (k + 3) * 2.0 ** -24)
    fi = torch.finfo(y.dtype)
    return out, bound + (out.abs() + bound) * fi.eps / 2 + fi.smallest_normal * fi.eps


def check_combine(dev, y, w, shared=None, gate=None):
    got = H.moe_combine(y.to(dev), w.to(dev), shared=None if shared is None else shared.to(dev),
                        shared_gate=None if gate is None else gate.to(dev))
    assert got.dtype == y.dtype and got.shape == (w.shape[0], y.shape[-1])
    ref, bound = combine(y, w, shared, gate)
    g = got.cpu().to(F64)
    assert torch.equal(torch.isnan(g), torch.isnan(ref))
    fine = torch.isfinite(ref)
    assert torch.equal(g[~fine].nan_to_num(5.0), ref[~fine].nan_to_num(5.0))
    assert bool(((g - ref).abs()[fine] <= bound[fine]).all()), float(((g - ref).abs() / bound)[fine].max())
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,top_k,hidden", [(1, 1, 8), (1, 10, 2048), (3, 4, 7), (5, 1, 1), (64, 10, 2048), (33, 6, 2880),
                                                 (130, 3, 1025), (2, 65, 100), (9, 8, 4096), (700, 2, 264)])
def test_combine_sizes(dev, tokens, top_k, hidden, dtype):
    g = torch.Generator().manual_seed(hidden)
    y = torch.randn((tokens * top_k, hidden), generator=g).to(dtype)
    w = torch.rand((tokens, top_k), generator=g)
    shared, gate = torch.randn((tokens, hidden), generator=g).to(dtype), 3 * torch.randn((tokens, 1), generator=g)
    check_combine(dev, y, w)
    check_combine(dev, y, w, shared)
    check_combine(dev, y, w, shared, gate.to(dtype))
    check_combine(dev, y, w, shared, gate)


def test_combine_zero_weights_and_odd_values(dev):
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(7)
    y = torch.randn((4 * 3, 64), generator=g).to(BF16)
    w = torch.rand((4, 3), generator=g)
    w[1, 0] = w[2, 2] = 0.0
    w[3] = 0.0
    y[3], y[8], y[9:] = nan, inf, nan  # rows of weight zero
    check_combine(dev, y, w)
    y[0, 5], y[1, 6], y[2, 6] = inf, inf, -inf
    w[0, 1] = -w[0, 1]
    check_combine(dev, y, w)
    shared, gate = torch.randn((4, 64), generator=g).to(BF16), torch.tensor([inf, -inf, -200.0, 200.0])
    check_combine(dev, y, w, shared, gate)


def test_combine_layouts(dev):
    g = torch.Generator().manual_seed(8)
    y = torch.randn((20, 4, 96), generator=g).to(BF16)
    w = torch.rand((20, 4), generator=g)
    want = check_combine(dev, y.reshape(80, 96), w)
    assert torch.equal(H.moe_combine(y.to(dev), w.to(dev)), want)
    assert torch.equal(H.moe_combine(y.to(dev), w.to(dev).reshape(4, 5, 4)), want.reshape(4, 5, 96))
    assert torch.equal(H.moe_combine(y.to(dev)[7], w.to(dev)[7]), want[7])
    wide = torch.zeros((80, 200), dtype=BF16, device=dev)
    ww = torch.zeros((20, 9), device=dev)
    ww[:, 3:7] = w.to(dev)
    for at in (8, 3):
        wide[:, at:at + 96] = y.reshape(80, 96).to(dev)
        out = torch.full((20, 200), 5.0, dtype=BF16, device=dev)
        H.moe_combine(wide[:, at:at + 96], ww[:, 3:7], out=out[:, at:at + 96])
        assert torch.equal(out[:, at:at + 96], want)
        assert bool((out[:, :at] == 5).all()) and bool((out[:, at + 96:] == 5).all())
    # the shared rows written over, the gate read from a wider projection
    shared, proj = torch.randn((20, 96), generator=g).to(BF16).to(dev), torch.randn((20, 5), generator=g).to(BF16).to(dev)
    a = H.moe_combine(y.to(dev), w.to(dev), shared=shared, shared_gate=proj[:, 2:3])
    assert torch.equal(a, H.moe_combine(y.to(dev), w.to(dev), shared=shared, shared_gate=proj[:, 2]))
    assert torch.equal(a, H.moe_combine(y.to(dev), w.to(dev), shared=shared, shared_gate=proj[:, 2].contiguous(), out=shared))
    assert H.moe_combine(y.to(dev)[:0].reshape(0, 96), w.to(dev)[:0]).shape == (0, 96)


def test_route_experts_combine_in_one_graph(dev):
    """A routed block as it is used: router, gate/up/down products, weighted sum."""
    g = torch.Generator().manual_seed(9)
    T, E, k, D, I = 24, 16, 4, 512, 512
    words = [torch.randint(-2 ** 31, 2 ** 31 - 1, s, generator=g, dtype=torch.int64).to(torch.int32).to(dev)
             for s in ((E, I, D // 8), (E, I, D // 8), (E, D, I // 8))]
    sc = [(0.004 + 0.002 * torch.rand((E, n, K // 64), generator=g)).to(BF16).to(dev) for n, K in ((I, D), (I, D), (D, I))]
    bi = [(-8 * s.float()).to(BF16) for s in sc]
    x = torch.randn((T, D), generator=g).to(BF16).to(dev)
    logits = torch.randn((T, E), generator=g).to(BF16).to(dev)
    shared, gate = torch.randn((T, D), generator=g).to(BF16).to(dev), torch.randn((T, 1), generator=g).to(BF16).to(dev)

    def block():
        w, e = H.moe_route(logits, k, renormalize=True)
        h = H.gather_qmm_swiglu(x, words[0], sc[0], bi[0], words[1], sc[1], bi[1], e, x_row_div=k)
        y = H.gather_qmm(h, words[2], sc[2], bi[2], e)
        return H.moe_combine(y, w, shared=shared, shared_gate=gate), w, e, y

    block()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, w, e, y = block()
    for _ in range(3):
        x.copy_(torch.randn((T, D), generator=g).to(BF16))
        logits.copy_(torch.randn((T, E), generator=g).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((out, w, e, y), block()):
            assert torch.equal(a, b)
        rw, re = route(logits.cpu(), k, renormalize=True)
        assert torch.equal(e.cpu(), re)
        ref, bound = combine(y.cpu(), w.cpu(), shared.cpu(), gate.cpu())
        assert bool(((out.cpu().to(F64) - ref).abs() <= bound).all())


def test_rows_far_apart(dev):
    """Rows beyond 2^31 elements of each other."""
    g = torch.Generator().manual_seed(10)
    far = torch.empty((20 << 27) + 512, dtype=BF16, device=dev)
    rows = far.as_strided((20, 128), (1 << 27, 1))
    x = torch.randn((20, 128), generator=g).to(BF16)
    rows.copy_(x)
    w, e = H.moe_route(rows, 6, renormalize=True)
    rw, re = route(x, 6, renormalize=True)
    assert torch.equal(e.cpu(), re) and float((w.cpu().to(F64) - rw).abs().max()) < 1e-5
    w = torch.rand((5, 4), generator=g)
    want = check_combine(dev, x, w)
    out = far.as_strided((5, 128), (5 << 27, 1), 256)
    assert torch.equal(H.moe_combine(rows, w.to(dev), out=out), want)


def test_on_another_stream(dev):
    """Work goes to the current stream, behind what is on it."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn((400, 256), generator=g).to(BF16)
    y = torch.randn((400 * 4, 512), generator=g).to(BF16)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        xd, yd = x.to(dev, non_blocking=True), y.to(dev, non_blocking=True)
        w, e = H.moe_route(xd, 4, renormalize=True)
        out = H.moe_combine(yd, w)
    s.synchronize()
    rw, re = route(x, 4, renormalize=True)
    assert torch.equal(e.cpu(), re)
    ref, bound = combine(y, w.cpu())
    assert bool(((out.cpu().to(F64) - ref).abs() <= bound).all())
