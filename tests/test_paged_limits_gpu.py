"""Paged attention where the sizes are unlike a usual step's.  Tolerance as in test_paged_gpu.py."""

import pytest
import torch

from xb200 import ops

pytestmark = pytest.mark.gpu


def _pool(positions, KVH, page, seed):
    """K and V of one sequence on the device: pages in reverse order, and the page table [1, columns]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = positions // page
    k, v = (torch.randn((n, KVH, page, 64), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    return k, v, torch.arange(n - 1, -1, -1, dtype=torch.int32, device="cuda").view(1, n)


@pytest.mark.parametrize("n,H,KVH,kv_len", [(200_000, 14, 2, 1024), (200_000, 28, 4, 1024), (95_000, 128, 1, 8192),
                                            (200_000, 14, 2, 0)])
def test_many_more_new_tokens_than_keys(n, H, KVH, kv_len):
    """Rows without a key are zeros and the last kv_len rows right; so is a short sequence beside it."""
    page, few = 16, 3
    k, v, table = _pool(max(kv_len, 1024) // page * page, KVH, page, n + H)
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn((n + few, H, 64), generator=g, device="cuda").to(torch.bfloat16)
    out = torch.full((n + few, H * 64), 7.0, dtype=torch.bfloat16, device="cuda")
    starts = torch.tensor([0, n, n + few], dtype=torch.int32, device="cuda")
    lens = torch.tensor([kv_len, 40], dtype=torch.int32, device="cuda")
    ops.paged_attention(q, k, v, out, table.repeat(2, 1), starts, lens, 0.125)
    out = out.view(-1, H, 64)
    assert bool((out[:n - kv_len] == 0).all())
    keys, values = (x[table[0].long()].transpose(1, 2).reshape(-1, KVH, 64).double() for x in (k, v))
    for lo, hi, length in ((n - kv_len, n, kv_len), (n, n + few, 40)):
        pos = length - (hi - lo) + torch.arange(hi - lo, device="cuda")
        for h in range(0, H, 5):
            s = q[lo:hi, h].double() @ keys[:length, h // (H // KVH)].T * 0.125
            p = torch.softmax(s.masked_fill(torch.arange(length, device="cuda") > pos[:, None], -torch.inf), -1)
            x = values[:length, h // (H // KVH)]
            want = p @ x
            bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * (p @ x.abs())
            assert bool(((out[lo:hi, h].double() - want).abs() <= bound).all())
    assert ops.device_status() == 0 and ops.page_status() == 0


@pytest.mark.parametrize("H,new", [(8, 3), (32, 70)])
def test_a_million_sequences_most_of_them_empty(H, new):
    """The largest batch: tokens of the first, a middle and the last sequence (few rows, many rows)."""
    B, page, kv_len = 1 << 20, 16, 1000
    k, v, table = _pool(1024, 1, page, H)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn((3 * new, H, 64), generator=g, device="cuda").to(torch.bfloat16)
    counts = torch.zeros(B + 1, dtype=torch.int64, device="cuda")
    counts[[1, B // 2 + 1, B]] = new
    starts = counts.cumsum(0).to(torch.int32)
    lens = torch.full((B,), kv_len, dtype=torch.int32, device="cuda")
    out = torch.full((3 * new, H * 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention(q, k, v, out, table.repeat(B, 1), starts, lens, 0.125)
    keys, values = (x[table[0].long()].transpose(1, 2).reshape(-1, 64).double()[:kv_len] for x in (k, v))
    pos = kv_len - new + torch.arange(new, device="cuda")
    s = q.double().view(3, new, H, 64).transpose(1, 2) @ keys.T * 0.125
    p = torch.softmax(s.masked_fill(torch.arange(kv_len, device="cuda") > pos[:, None], -torch.inf), -1)
    want, a = ((p @ x).transpose(1, 2).reshape(3 * new, -1) for x in (values, values.abs()))
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * a).all())
    assert ops.device_status() == 0 and ops.page_status() == 0


def test_copies_of_pages_of_half_a_gigabyte():
    """As a cache with pages of 2^20 positions of four heads has them: 500 would pass a launch's 2^32 vectors."""
    g = torch.Generator(device="cuda").manual_seed(3)
    pool = torch.randint(0, 1 << 30, (2, 5, 1 << 27), dtype=torch.int32, generator=g, device="cuda")
    want = pool[:, :2].clone()
    last = pool[:, 4].clone()
    assert ops.copy_pages(pool, [0, 1], [3, 2], dim=1) is pool
    for at, page in ((0, want[:, 0]), (1, want[:, 1]), (3, want[:, 0]), (2, want[:, 1]), (4, last)):
        assert torch.equal(pool[:, at], page)
