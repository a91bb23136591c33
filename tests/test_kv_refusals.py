"""Refusals of the paged cache's calls, on the CPU: every call gives the status
of its reason."""
from __future__ import annotations

import pytest
import torch

import higgs_amd as H
from higgs_amd._lib import HgkError


@pytest.mark.parametrize("dtype,head_dim", [(torch.float32, 64), (torch.bfloat16, 80), (torch.float16, 512)])
def test_what_is_not_supported_says_so(dtype, head_dim):
    """Types and head sizes that no kernel is for: status 2."""
    p = torch.zeros((4, 16, 2, head_dim), dtype=dtype)
    q = torch.zeros((2, 4, head_dim), dtype=dtype)
    t, n = torch.zeros((2, 3), dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(HgkError) as e:
        H.paged_attention(q, p, p, t, n)
    assert e.value.status == 2
    # sizes that are wrong and not unsupported keep status 1
    q = torch.zeros((2, 3, 64), dtype=torch.bfloat16)
    p = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(HgkError, match="heads") as e:
        H.paged_attention(q, p, p, t, n)
    assert e.value.status == 1


def test_a_sequence_ends_where_a_table_does():
    """2^30 tokens are the most that a call's table holds: no pages are given out beyond."""
    c = H.PagedKVCache(1, 2 ** 14 + 1, 65536, 1, 64, device="meta")
    a = c.new()
    c.extend([a], [2 ** 30 - 5])
    for n in (6, 2 ** 31):
        with pytest.raises(HgkError, match="2\\^30"):
            c.extend([a], [n])
    assert c.length(a) == 2 ** 30 - 5 and c.free_pages == 1
    c.extend([a], [5])
    assert c.length(a) == 2 ** 30


def append(k_pages, v_pages, k, v):
    """hgk_kv_append's status and message for a call of 2^30 rows, which it refuses
    for their number if for nothing else: no kernel is launched."""
    import ctypes as C

    from higgs_amd import _lib, ops
    from higgs_amd._lib import HgkKvBatch

    fake, what, L = 1 << 20, "kv_append", _lib.lib()
    b = HgkKvBatch(batch=1, tokens=1 << 30, block_table=fake, table_stride=4, table_width=4, kv_lens=fake, q_starts=fake)
    s = L.hgk_kv_append(ops._pool(k_pages, v_pages, what), C.byref(b), k.data_ptr(),
                        ops._token_rows(k, k_pages, what, "k"), v.data_ptr(), ops._token_rows(v, k_pages, what, "v"),
                        None)
    return s, L.hgk_last_error().decode()


def test_key_pages_on_value_pages():
    """Two rows that a call writes to one place: the last write would win by chance."""
    pool = torch.zeros((9, 2, 16, 2, 64), dtype=torch.bfloat16)
    k, v = (torch.zeros((2, 2, 64), dtype=torch.bfloat16) for _ in range(2))
    flat = pool.view(18, 16, 2, 64)
    for kp, vp in ((flat, flat), (flat[:9], flat[1:10]), (flat[:9], flat[8:17]), (pool[:, 0], pool[:, 0]),
                   (pool[:8, 0], pool[1:, 0]), (flat[:, :8], flat[:, 4:12])):
        s, msg = append(kp, vp, k, v)
        assert s == 1 and "overlap" in msg, (kp.stride(), msg)
    # side by side in every way that a pool is cut
    heads = torch.zeros((9, 16, 4, 64), dtype=torch.bfloat16)
    wide = torch.zeros((9, 16, 2, 128), dtype=torch.bfloat16)
    other = torch.zeros((18, 16, 2, 64), dtype=torch.bfloat16)
    for kp, vp in ((pool[:, 0], pool[:, 1]), (pool[:, 1], pool[:, 0]), (flat[:9], flat[9:]), (flat[9:], flat[:9]),
                   (flat[::2], flat[1::2]), (heads[:, :, :2], heads[:, :, 2:]), (heads[:, :, ::2], heads[:, :, 1::2]),
                   (wide[..., :64], wide[..., 64:]), (flat, other), (flat[:, :8], flat[:, 8:])):
        assert "too many" in append(kp, vp, k, v)[1], kp.stride()
    assert "too many" in append(flat, flat, k, k)[1]  # keys that are the values
