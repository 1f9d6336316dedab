"""8-bit pages where sizes are unlike a usual step's.  Tolerances as in test_paged8_gpu.py."""

import pytest
import torch
from test_paged8_gpu import DTYPES, Coded

from xb200 import ops

pytestmark = pytest.mark.gpu


def _far(b, stride):
    """The same batch with `stride` bytes between pages: the last ones lie behind 2^32 bytes."""
    n, KVH, P, D = b.kp.shape
    for name in ("kp", "vp"):
        flat = torch.empty((n - 1) * stride + KVH * P * D, dtype=torch.uint8, device="cuda")
        far = flat.as_strided((n, KVH, P, D), (stride, P * D, D, 1))
        far.copy_(getattr(b, name).view(torch.uint8))
        setattr(b, name, far.view(b.dtype))
    step = stride // 2
    for name in ("ks", "vs"):
        flat = torch.empty((n - 1) * step + KVH * P, dtype=torch.uint8, device="cuda")
        far = flat.as_strided((n, KVH, P), (step, P, 1))
        far.copy_(getattr(b, name))
        setattr(b, name, far)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1, 1], [60, 1, 40]])
def test_pools_of_more_than_2_32_bytes(new, dtype):
    b = Coded(dtype, new, [30, 190, 11], 14, 2, 16, seed=60)
    want = b.attend()
    _far(b, 2 ** 29)
    assert int(b.table.max()) * 2 ** 29 > 2 ** 32 and torch.equal(b.attend(), want)
    counts = [x.shape[0] for x in b.k]
    starts = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()
    k, v = (torch.empty((sum(counts), 2, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.paged_read_kv(k, v, b.kp, b.vp, b.table_dev, starts, b.kv_len, b.ks, b.vs)
    assert torch.equal(k.cpu().double(), torch.cat(b.k)) and torch.equal(v.cpu().double(), torch.cat(b.v))
    # what is read back is written again: the same values (a largest code that was rounded down may take another exponent)
    qkv = torch.cat([torch.zeros((len(k), 14 * 64), dtype=torch.bfloat16, device="cuda"), k.flatten(1), v.flatten(1)], 1)
    b.ks.fill_(255), b.vs.fill_(255)
    q = torch.empty((len(k), 14, 64), dtype=torch.bfloat16, device="cuda")
    ops.paged_rope_kv(qkv, None, None, q, b.kp, b.vp, b.table_dev, starts, b.kv_len, b.ks, b.vs)
    k.fill_(7), v.fill_(7)
    ops.paged_read_kv(k, v, b.kp, b.vp, b.table_dev, starts, b.kv_len, b.ks, b.vs)
    assert torch.equal(k.cpu().double(), torch.cat(b.k)) and torch.equal(v.cpu().double(), torch.cat(b.v))
    b.check(b.attend())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,cols", [([1] * 70, 300_000), ([2] * 30, 300_000), ([200, 1, 57], 1000)])
def test_wide_tables(new, cols, dtype):
    """64-bit walks of the few-row kernel; a pool smaller than the table for the many-row one."""
    b = Coded(dtype, new, [37 * i % 613 for i in range(len(new))], 14, 2, 16, seed=61)
    wide = torch.full((len(new), cols), -1, dtype=torch.int32, device="cuda")
    wide[:, :b.table.shape[1]] = b.table_dev
    narrow, b.table_dev = b.table_dev, wide
    out = b.attend()
    b.check(out)
    b.table_dev = narrow
    b.check(b.attend())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KVH", [(14, 2), (16, 1), (12, 12)])
def test_where_the_two_tile_sizes_meet(H, KVH, dtype):
    """Tables for just under and just over 96 keys a warp of 148 SMs: tiles of 32 and of 64 keys."""
    border = 96 * 8 * 148 // (5 * KVH * 16)
    for cols in (border, border + 1):
        b = Coded(dtype, [1] * 5, [1700, 64, 1, 0, 129], H, KVH, 16, seed=62)
        wide = torch.zeros((5, cols), dtype=torch.int32, device="cuda")
        wide[:, :min(cols, b.table.shape[1])] = b.table_dev[:, :cols].clamp(min=0)
        b.table_dev = wide
        b.check(b.attend())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,H,KVH", [([1] * 11, 14, 2), ([1] * 12, 14, 2), ([1] * 74, 14, 2), ([1] * 75, 14, 2),
                                       ([2, 0, 5, 1], 14, 2), ([1, 3, 2], 12, 12), ([16, 1, 9], 4, 4), ([1] * 148, 8, 1),
                                       ([1], 16, 1)])
def test_where_units_have_a_cta_each(new, H, KVH, dtype):
    """Tables of two and three tiles a warp (8 or 12 of them), and of one page more; lengths from none to all of them."""
    g = torch.Generator().manual_seed(90)
    for positions in (512, 528, 768, 784, 1152, 1168):
        lens = [int(x) for x in torch.randint(0, positions, (len(new),), generator=g)]
        lens[-1] = positions  # all of it
        lens[0] = 1
        b = Coded(dtype, new, [x - n for x, n in zip(lens, new)], H, KVH, 16, seed=91, pad=2)
        table = torch.full((len(new), positions // 16), -1, dtype=torch.int32, device="cuda")
        table[:, :b.table.shape[1]] = b.table_dev
        b.table_dev = table
        out = b.attend()
        b.check(out)
        assert bool((out[-2:] == 7).all()) and torch.equal(out, b.attend())


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences_without_a_key(dtype):
    b = Coded(dtype, [70] + [1] * 600 + [9] + [1] * 600, [100] + [-1] * 600 + [300] + [-1] * 600, 32, 1, 16, seed=63)
    out = b.attend()
    b.check(out)
    assert bool((out[70:670] == 0).all()) and bool((out[679:] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,new", [(8, 3), (32, 70)])
def test_a_million_sequences_most_of_them_empty(H, new, dtype):
    small = Coded(dtype, [new] * 3, [1000 - new] * 3, H, 1, 16, seed=64)
    B = 1 << 20
    at = torch.tensor([0, B // 2, B - 1])
    counts = torch.zeros(B + 1, dtype=torch.int64)
    counts[at + 1] = new
    starts = counts.cumsum(0).to(torch.int32).cuda()
    lens = torch.full((B,), 1000, dtype=torch.int32, device="cuda")
    table = torch.full((B, small.table.shape[1]), -1, dtype=torch.int32, device="cuda")
    table[at] = small.table_dev
    want = small.attend()
    small.check(want)
    small.q_start, small.kv_len, small.table_dev = starts, lens, table
    small.check(small.attend())
    k, v = (torch.empty((3 * new, 1, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.paged_read_kv(k, v, small.kp, small.vp, table, starts, lens, small.ks, small.vs)
    assert torch.equal(k.cpu().double(), torch.cat([x[-new:] for x in small.k]))
    qkv = torch.cat([torch.zeros((3 * new, H * 64), dtype=torch.bfloat16, device="cuda"), k.flatten(1), v.flatten(1)], 1)
    q = torch.full((3 * new, H, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_rope_kv(qkv, None, None, q, small.kp, small.vp, table, starts, lens, small.ks, small.vs)
    small.check(small.attend())
    assert bool((q == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,KVH,kv_len", [(20_000, 14, 2, 1024), (20_000, 14, 2, 0)])
def test_many_more_new_tokens_than_keys(n, H, KVH, kv_len, dtype):
    b = Coded(dtype, [n, 3], [kv_len - n, 37], H, KVH, 16, seed=65)
    out = b.attend()
    assert bool((out[:n - kv_len] == 0).all())
    rows = slice(n - kv_len, n + 3)
    b.q, b.T, b.new, b.starts = b.q[rows], kv_len + 3, [kv_len, 3], [0, kv_len, kv_len + 3]
    b.check(out[rows])


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_beyond_the_table_are_cut_and_ranges_clamped(dtype):
    b = Coded(dtype, [1, 1], [63, 20], 14, 2, 16, seed=66)
    want = b.attend()
    b.kv_len[0] = 2 ** 31 - 1  # the table holds 64 positions
    assert torch.equal(b.attend(), want)
    b.kv_len[1] = -5
    assert bool((b.attend()[1] == 0).all())
    b.kv_len[1] = 21
    for starts in ([-7, 1, 1 << 30], [5, 2, 0]):
        b.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        b.attend()
    c = Coded(dtype, [40, 60], [30, 500], 14, 2, 16, seed=67)
    c.kv_len[0] = 2 ** 31 - 1
    c.attend()
    c.q_start.copy_(torch.tensor([90, 2, 0], dtype=torch.int32))
    assert bool((c.attend() == 7).all())  # descending: nothing belongs to anyone
    assert ops.device_status() == 0
    ops.page_status()


@pytest.mark.parametrize("dtype", DTYPES)
def test_calls_from_several_threads(dtype):
    import threading

    batches = [Coded(dtype, [1] * 5, [300, 9, 77, 0, 1200], 14, 2, 16, seed=68),
               Coded(dtype, [150, 2], [30, 500], 12, 12, 32, seed=69)]
    qs, want = [b.q.cuda() for b in batches], [b.attend() for b in batches]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(batches[i % 2].attend(qs[i % 2]), want[i % 2]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and ops.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_attention_and_reading_back_in_one_graph(dtype):
    """Captured once, replayed for other tokens at other positions of other pages."""
    b = Coded(dtype, [1, 3], [40, 20], 14, 2, 16, seed=70, extra_cols=2)
    qkv = torch.randn((4, 18 * 64), generator=torch.Generator().manual_seed(71)).to(torch.bfloat16).cuda()
    q, out = (torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in ((4, 14, 64), (4, 14 * 64)))
    k, v = (torch.empty((4, 2, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def step():
        ops.paged_rope_kv(qkv, None, None, q, b.kp, b.vp, b.table_dev, b.q_start, b.kv_len, b.ks, b.vs)
        b.attend(q, out)
        ops.paged_read_kv(k, v, b.kp, b.vp, b.table_dev, b.q_start, b.kv_len, b.ks, b.vs)

    step()
    first = [x.clone() for x in (out, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(first, (out, k, v)))
    qkv.mul_(3)
    b.table_dev.copy_(b.table_dev.flip(0))
    b.kv_len.copy_(torch.tensor([10, 39], dtype=torch.int32))
    b.q_start.copy_(torch.tensor([0, 2, 4], dtype=torch.int32))
    graph.replay()
    got = [x.clone() for x in (q, out, k, v)]
    for x in (q, out, k, v):
        x.fill_(7)
    step()
    assert all(torch.equal(x, y) for x, y in zip(got, (q, out, k, v))) and ops.page_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,H,KVH", [([6, 4], 4, 4), ([12, 16], 4, 4), ([3, 2], 14, 2), ([40, 70], 14, 2)])
def test_nan_of_a_new_token_leaves_the_earlier_ones(new, H, KVH, dtype):
    """What a token writes, those before it in the same step do not see: 8 and 16 rows, and the expanded pages."""
    b = Coded(dtype, new, [30, 75], H, KVH, 16, seed=72)
    clean = b.attend().view(b.T, KVH, -1)
    for pool, scale in ((b.kp, b.ks), (b.vp, b.vs)):
        for i, at in ((0, new[0] - 1), (1, new[1] // 2), (1, 0)):
            p = b.k[i].shape[0] - new[i] + at
            page, row = int(b.table[i, p // 16]), p % 16
            was = pool[page, 0, row].clone(), scale[page, 0, row].clone()
            pool[page, 0, row], scale[page, 0, row] = 0, 255
            out = b.attend().view(b.T, KVH, -1)
            bad = torch.isnan(out)
            sees = torch.zeros((b.T, KVH, 1), dtype=torch.bool, device="cuda")
            sees[b.starts[i] + at:b.starts[i + 1], 0] = True
            assert torch.equal(bad, sees.expand_as(bad))
            b.check(torch.where(bad, clean, out).view(b.T, -1))  # a lost maximum may move the others' base
            pool[page, 0, row], scale[page, 0, row] = was
