"""moe_route where scores are below what f32 holds, against the definition in 64 bits.

Counted as in test_gpu_moe.py: a weight is within (2 * 2^-22 + (n + top_k + 6) 2^-24) of
itself; 2^-24 of how far its logit is below the one that it is taken from, whose difference
is rounded once (of the others' in a sum no more than 0.4 each counts: x e^-x); and half
a step of f32's least, 2^-150, for each of the score, the quotient and the product with the
scale (which the scale multiplies)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import higgs_amd as H

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def expected(x, experts, scores, renormalize, scale):
    """(weights of the experts given, the logs of the scores first; how far the logits are below)."""
    l = x.to(F64).numpy()
    chosen = np.take_along_axis(l, experts.numpy().astype(np.int64), 1)
    most = (chosen if renormalize else l).max(1, keepdims=True)
    below = (most if scores == "softmax" else np.minimum(most, 0.0) if renormalize else 0.0 * most) - chosen
    if scores == "softmax":
        s = l - (l.max(1, keepdims=True) + np.log(np.exp(l - l.max(1, keepdims=True)).sum(1, keepdims=True)))
    else:
        s = -np.logaddexp(0.0, -l)
    s = np.take_along_axis(s, experts.numpy().astype(np.int64), 1)
    none = s.max(1, keepdims=True) < -750  # no score in 64 bits either: zeros
    if renormalize:
        s = s - (s.max(1, keepdims=True) + np.log(np.exp(s - s.max(1, keepdims=True)).sum(1, keepdims=True)))
    return torch.tensor(np.where(none, 0.0, np.exp(s)) * scale), torch.tensor(np.maximum(below, 0.0))


def check(dev, x, top_k, bias=None, scores="softmax", renormalize=True, scale=1.0, **kw):
    w, e = H.moe_route(x.to(dev), top_k, scores=scores, renormalize=renormalize, scale=scale,
                       bias=None if bias is None else bias.to(dev), **kw)
    w, e = w.cpu().to(F64), e.cpu()
    ref, below = expected(x, e, scores, renormalize, scale)
    bound = ref * (2 * 2.0 ** -22 + (x.shape[1] + top_k + 6 + below) * 2.0 ** -24) + 3 * max(scale, 1.0) * 2.0 ** -150
    assert bool(((w - ref).abs() <= bound).all()), (w[0], ref[0])
    if renormalize:
        assert bool(((w.sum(1) - scale * (ref.sum(1) > 0)).abs() <= scale * 2.0 ** -20).all())
    return e


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("experts", [8, 70, 256, 1024])
@pytest.mark.parametrize("at", [-70.0, -90.0, -105.0, -200.0, -3000.0])
def test_sigmoids_of_logits_far_below_zero(dev, at, experts, dtype):
    g = torch.Generator().manual_seed(21)
    x = (at + 3 * torch.randn((6, experts), generator=g)).to(dtype)
    check(dev, x, 5, scores="sigmoid")
    check(dev, x, 5, scores="sigmoid", scale=2.5)
    check(dev, x, 5, scores="sigmoid", bias=torch.rand((experts,), generator=g))
    x[:, 3] = at - 60
    x[0, 0] = 0.5  # one above zero beside them
    check(dev, x, 8, scores="sigmoid")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("below", [20.0, 88.0, 100.0, 104.0, 300.0])
def test_experts_that_a_bias_puts_in_front(dev, below, dtype):
    """Chosen experts whose logits are `below` the row's greatest."""
    g = torch.Generator().manual_seed(22)
    x = torch.randn((7, 128), generator=g)
    x[:, 10:16] -= below
    x = x.to(dtype)
    bias = torch.zeros(128)
    bias[10:16] = 5.0 + torch.arange(6)
    e = check(dev, x, 6, bias=bias)
    assert bool(((e >= 10) & (e < 16)).all())
    check(dev, x, 6, bias=bias, scale=1e20)
    e = check(dev, x, 4, bias=bias, groups=8, top_groups=1, group_top=2)
    assert bool(((e >= 10) & (e < 16)).all())
    check(dev, x, 6, bias=bias, renormalize=False)
    check(dev, x, 6, bias=bias, renormalize=False, scale=2.0 ** 60)


@pytest.mark.parametrize("at", [-86.0, -90.0, -100.0, -103.0])
def test_scores_among_the_least_that_f32_holds(dev, at):
    g = torch.Generator().manual_seed(23)
    x = at + torch.rand((9, 64), generator=g)
    check(dev, x, 8, scores="sigmoid", renormalize=False)
    x[:, 0] = 0.0
    check(dev, x, 8, renormalize=False)
    check(dev, x, 8, renormalize=True)


def test_rows_that_hold_no_score(dev):
    """Renormalising leaves zeros where no chosen expert has any."""
    inf = float("inf")
    x = torch.full((4, 16), -inf)
    x[1, 3] = inf
    x[2, 3] = -500.0
    x[3, 3] = inf
    bias = torch.zeros(16)
    bias[5:9] = 9.0
    for scores in ("softmax", "sigmoid"):
        w, _ = H.moe_route(x.to(dev), 4, scores=scores, renormalize=True)
        assert torch.equal(w.cpu(), torch.tensor([[0.0] * 4, [1.0, 0, 0, 0], [1.0, 0, 0, 0], [1.0, 0, 0, 0]]))
        w, e = H.moe_route(x.to(dev), 4, scores=scores, renormalize=True, bias=bias.to(dev))
        assert torch.equal(e.cpu(), torch.arange(5, 9, dtype=torch.int32).expand(4, 4)) and bool((w == 0).all())
