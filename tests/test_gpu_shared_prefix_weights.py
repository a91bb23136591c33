"""Single tokens' weights keep two 16-bit parts with and without a pass over the prefix, so
that a row is as exact whoever else is in its batch.

Counted as in kv_ref.py, but for the weights: of a half step u each part leaves at most u of
what it rounds, so both leave u^2 of a weight, and their sum as much: 2 u^2 in place of u.

The errors of a whole result, next to those of the exact one rounded once: of rounding alone
they are some 0.4 u of an element (2^-12.3 in f16), and the f32 scores' and exponents' errors
of 2^-20 at the most, over many keys, add nothing to their sum of squares that shows. Weights in
one part made it 1.37 times as great a norm; 1.1 is held."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
import kv_ref as R
from test_gpu_shared_prefix import BF16, F16, call, lens_of, make, many

pytestmark = pytest.mark.gpu


def check(got, y, what="", **kw):
    out, bound, owned = R.reference(y, **kw)
    mag = R.attend(y["q"], y["k_pages"], y["v_pages"].abs(), y["table"], y["lens"], y["starts"], **kw)[0]
    u = torch.finfo(got.dtype).eps / 2
    R.check(got, (out, (bound - mag * (u - 2 * u * u)) * (1 + u), owned), what)
    rounded = (out.to(got.dtype).to(R.F64) - out).norm()
    assert float((got.to(R.F64) - out).norm()) <= 1.1 * float(rounded), what


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(32, 8, 64), (32, 8, 128), (16, 2, 256), (4, 1, 96), (40, 1, 64)])
def test_rows_behind_a_pass(dev, heads, kv_heads, head_dim, dtype):
    prefix = 1501
    lens, _ = lens_of(prefix, many(prefix, kv_heads, head_dim), False)
    lens[0], lens[1] = 700, 0  # some of the prefix, none of it
    x, y = make(81, prefix, lens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=16, dtype=dtype)
    check(call(R.to(x, dev), prefix).cpu(), y)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("softcap", [0.0, 50.0, 200.0])
def test_windows_and_caps(dev, softcap, head_dim, dtype):
    """Tiles that some row sees in part, and soft caps."""
    prefix = 1400
    lens, _ = lens_of(prefix, 2 * many(prefix, 4, head_dim), False, 300)
    x, y = make(82, prefix, lens, heads=8, kv_heads=4, head_dim=head_dim, page=16, dtype=dtype, q_scale=2.0)
    d = R.to(x, dev)
    for kw in ({}, {"window": 1300, "sinks": 70}):
        check(call(d, prefix, softcap=softcap, **kw).cpu(), y, str(kw), softcap=softcap, **kw)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_as_exact_in_a_batch_of_two(dev, dtype):
    """The same sequences in a batch that is not worth a pass, and over tables of their own."""
    prefix = 1501
    lens, _ = lens_of(prefix, many(prefix, 8, 128), False)
    x, y = make(83, prefix, lens, heads=32, kv_heads=8, head_dim=128, page=16, dtype=dtype)
    for z in (x, y):
        for name in ("q", "table", "lens"):
            z[name] = z[name][:2].clone()
    check(call(R.to(x, dev), prefix).cpu(), y)
    check(R.call(H, R.to(y, dev)).cpu(), y)
