"""The paged KV cache's operators against plain 64-bit implementations.

Every page no sequence uses, and every row behind a sequence's last position,
holds NaN: whatever a kernel reads there must not reach a result.

Tolerance of the attention, per element: the result is rounded to bf16 once
(half a step: 2^-8 of its value), and each weight is rounded to bf16 before it
multiplies its value (2^-8 of the weighted sum of |v|); fp32 scores,
exponentials and sums add less than 2^-12 of that sum (a score of magnitude
up to 64 carries 2^-18, the exponential's argument the same).
"""

import math
import random

import pytest
import torch

from oracle import qwen as OQ
from xb200 import ops

pytestmark = pytest.mark.gpu

NAN = float("nan")


class Batch:
    """A ragged batch over a poisoned pool; kv_len[b] = past[b] + new[b]."""

    def __init__(self, new, past, H, KVH, page, seed=0, layout="nhpd", pad=0, extra_cols=0, D=64):
        g = torch.Generator().manual_seed(seed)
        rnd = random.Random(seed)
        self.new, self.past, self.H, self.KVH, self.page, self.D = new, past, H, KVH, page, D
        B = len(new)
        length = [max(0, a + b) for a, b in zip(new, past)]
        used = [-(-x // page) for x in length]
        n = sum(used) + 3
        order = list(range(n))
        rnd.shuffle(order)
        cols = max(used + [1]) + extra_cols
        self.table = torch.full((B, cols), -1, dtype=torch.int32)  # unused columns name no page
        for b, u in enumerate(used):
            for i in range(u):
                self.table[b, i] = order.pop()
        self.k = [torch.randn((x, KVH, D), generator=g).mul(2).to(torch.bfloat16) for x in length]
        self.v = [torch.randn((x, KVH, D), generator=g).to(torch.bfloat16) for x in length]
        shape = (n, KVH, page, D)
        kp, vp = torch.full(shape, NAN, dtype=torch.bfloat16), torch.full(shape, NAN, dtype=torch.bfloat16)
        for b in range(B):
            for p in range(length[b]):
                i, r = self.table[b, p // page], p % page
                kp[i, :, r], vp[i, :, r] = self.k[b][p], self.v[b][p]
        if layout == "nhpd":
            self.kp, self.vp = kp.cuda(), vp.cuda()
        elif layout == "joint":  # K and V of a page side by side
            both = torch.stack([kp, vp], 1).cuda()
            self.kp, self.vp = both[:, 0], both[:, 1]
        elif layout == "rows":  # heads inside rows
            self.kp = kp.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
            self.vp = vp.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
        starts = [0]
        for x in new:
            starts.append(starts[-1] + x)
        self.T = starts[-1] + pad
        self.starts = starts
        self.q_start = torch.tensor(starts, dtype=torch.int32).cuda()
        self.kv_len = torch.tensor(length, dtype=torch.int32).cuda()
        self.table_dev = self.table.cuda()
        self.q = torch.randn((self.T, H, D), generator=g).mul(2).to(torch.bfloat16)

    def attend(self, q=None, out=None, scale=0.125):
        q = self.q.cuda() if q is None else q
        if out is None:
            out = torch.full((self.T, self.H * self.D), 7.0, dtype=torch.bfloat16, device="cuda")
        return ops.paged_attention(q, self.kp, self.vp, out, self.table_dev, self.q_start, self.kv_len, scale)

    def exact(self, scale=0.125):
        """(o, sum of p |v|) in 64 bits; rows outside the sequences NaN in the second."""
        o = torch.full((self.T, self.H, self.D), 7.0, dtype=torch.float64)
        a = torch.zeros((self.T, self.H, self.D), dtype=torch.float64)
        rep = self.H // self.KVH
        for b, n in enumerate(self.new):
            t = self.starts[b]
            k = self.k[b].double().repeat_interleave(rep, 1).transpose(0, 1)  # [H, L, D]
            v = self.v[b].double().repeat_interleave(rep, 1).transpose(0, 1)
            L = k.shape[1]
            pos = L - n + torch.arange(n)
            s = self.q[t:t + n].double().transpose(0, 1) @ k.transpose(1, 2) * scale
            s = s.masked_fill(torch.arange(L)[None, :] > pos[:, None], -math.inf)
            p = torch.softmax(s, -1)
            p[:, pos < 0] = 0.0  # no key: zeros
            o[t:t + n] = (p @ v).transpose(0, 1)
            a[t:t + n] = (p @ v.abs()).transpose(0, 1)
        return o, a

    def check(self, out, scale=0.125):
        o, a = self.exact(scale)
        got = out.cpu().double().reshape(self.T, self.H, self.D)
        assert bool(torch.isfinite(got).all())
        bound = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -12) * a
        over = (got - o).abs() - bound
        assert float(over.max()) <= 0.0 if over.numel() else True, (float(over.max()), int(over.argmax()))
        assert ops.device_status() == 0 and ops.page_status() == 0


SHAPES = [
    # new tokens, earlier positions, H, KVH, page
    ([1], [0], 14, 2, 16),  # one token, one key
    ([1], [511], 14, 2, 16),
    ([1] * 9, [0, 1, 14, 15, 16, 31, 32, 33, 700], 14, 2, 16),  # around page and tile ends
    ([1] * 70, [37 * i % 613 for i in range(70)], 14, 2, 16),
    ([1] * 5, [5000, 3, 0, 129, 2047], 12, 12, 32),  # one long context among short ones
    ([1] * 3, [100, 7, 300], 16, 1, 64),
    ([1, 0, 1, 0, 0, 1, 0], [5, 9, 40, 0, 77, 64, 3], 14, 2, 16),  # sequences without new tokens
    ([2, 5, 1, 3], [30, 31, 0, 250], 14, 2, 16),
    ([7, 1, 12], [0, 64, 20], 4, 4, 8),
    ([33, 1, 64], [0, 90, 17], 9, 3, 48),
    ([100], [0], 14, 2, 16),
    ([130, 1, 257, 64], [0, 333, 70, 0], 14, 2, 16),
    ([300, 5], [37, 1000], 12, 12, 64),
    ([128, 127, 129], [0, 1, 128], 25, 25, 16),
    ([40], [3000], 32, 8, 128),
    ([1] * 300, [i % 50 for i in range(300)], 10, 2, 16),  # more sequences than threads
    ([3] * 260, [(i * 7) % 90 for i in range(260)], 20, 4, 8),
    ([513], [2000], 14, 2, 64),
]


@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_matches_64_bits(case):
    new, past, H, KVH, page = SHAPES[case]
    b = Batch(new, past, H, KVH, page, seed=case)
    out = b.attend()
    b.check(out)
    assert torch.equal(out, b.attend())  # joined in a fixed order


@pytest.mark.parametrize("layout", ["joint", "rows"])
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 1, 200]])
def test_attention_over_strided_pages_and_pitched_rows(layout, new):
    b = Batch(new, [40, 513, 3], 14, 2, 16, seed=3, layout=layout, extra_cols=5)
    wide = torch.zeros((b.T, 18 * 64), dtype=torch.bfloat16, device="cuda")
    q = wide[:, :14 * 64].view(b.T, 14, 64)
    q.copy_(b.q)
    wide_out = torch.full((b.T, 16 * 64), 7.0, dtype=torch.bfloat16, device="cuda")
    b.attend(q, wide_out[:, 64:15 * 64])
    b.check(wide_out[:, 64:15 * 64])
    assert bool((wide_out[:, :64] == 7).all()) and bool((wide_out[:, 15 * 64:] == 7).all())


@pytest.mark.parametrize("new", [[1, 1], [90, 3]])
def test_rows_behind_the_last_sequence_stay(new):
    b = Batch(new, [20, 30], 14, 2, 16, seed=4, pad=5)
    out = b.attend()
    b.check(out)
    assert bool((out[-5:] == 7).all())


@pytest.mark.parametrize("new,past", [([4, 1], [-2, 10]), ([1, 2], [-1, -2]), ([150, 20], [-140, 5])])
def test_tokens_without_a_key_get_zeros(new, past):
    """kv_len below the number of new tokens: the first tokens have no position."""
    b = Batch(new, past, 14, 2, 16, seed=5)
    out = b.attend()
    b.check(out)
    assert bool((out[:-past[0]] == 0).all())


def test_many_sequences_without_a_key():
    """Units without a key tile follow one with keys in the same share of work, more of them than a CTA looks ahead."""
    b = Batch([70] + [1] * 4000 + [9] + [1] * 4000, [100] + [-1] * 4000 + [300] + [-1] * 4000, 32, 1, 16, seed=50)
    out = b.attend()
    b.check(out)
    assert bool((out[70:4070] == 0).all()) and bool((out[4079:] == 0).all())


def test_infinite_and_nan_inputs_stay_in_their_rows():
    """A NaN query spoils its own rows only; a NaN key those that see it; a -inf score weighs nothing."""
    b = Batch([40, 1], [0, 30], 14, 2, 16, seed=6)
    b.q[3, 5, 0] = NAN
    clean = b.attend(torch.nan_to_num(b.q).cuda())
    out = b.attend()
    hit = torch.isnan(out.view(b.T, 14, 64)).any(-1).cpu()
    assert hit.nonzero().tolist() == [[3, 5]]
    b.q = torch.nan_to_num(b.q)
    b.check(torch.where(hit.cuda()[..., None], clean.view(b.T, 14, 64), out.view(b.T, 14, 64)))
    page, row = int(b.table[0, 1]), 4  # position 20 of sequence 0
    b.kp[page, 0, row, 0] = NAN
    bad = torch.isnan(b.attend().view(b.T, 2, 7 * 64)).any(-1).cpu()
    assert bad[:, 0].tolist() == [20 <= t < 40 for t in range(41)] and not bool(bad[:, 1].any())


def test_every_score_minus_infinity():
    """Keys of -inf in the sign of the query: scores of -inf weigh nothing, and rows with no other key are zeros."""
    b = Batch([3], [0], 1, 1, 16, seed=7)
    b.q = b.q.abs() + 1
    page = int(b.table[0, 0])
    b.kp[page, 0, 0] = -math.inf
    out = b.attend()
    assert bool((out[0] == 0).all())
    b.k[0][0] = 0
    k, v = b.k[0][1:, 0].double(), b.v[0][1:, 0].double()
    s = b.q[1:, 0].double() @ k.T * 0.125
    s[0, 1] = -math.inf
    p = torch.softmax(s, -1)
    bound = 2.0 ** -8 * (p @ v).abs() + (2.0 ** -8 + 2.0 ** -12) * (p @ v.abs())
    assert bool(((out[1:].cpu().double() - p @ v).abs() <= bound).all())


@pytest.mark.parametrize("new", [[1, 1, 1], [60, 1, 90]])
def test_bad_pages_read_as_zeros_and_are_reported(new):
    b = Batch(new, [100, 50, 200], 14, 2, 16, seed=8)
    assert ops.page_status() == 0
    for j, bad in ((0, -1), (2, b.kp.shape[0]), (3, 2 ** 31 - 1), (4, -2 ** 31)):
        b.table_dev[2, j] = bad
        lo = j * 16
        b.k[2][lo:lo + 16] = 0
        b.v[2][lo:lo + 16] = 0
    out = b.attend()
    assert ops.page_status() == 1
    b.check(out)  # the flag is clear again


def test_lengths_beyond_the_table_are_cut():
    b = Batch([1, 1], [63, 20], 14, 2, 16, seed=9)
    want = b.attend()
    b.kv_len[0] = 2 ** 31 - 1  # the table holds 64 positions
    assert torch.equal(b.attend(), want)
    b.kv_len[1] = -5
    assert bool((b.attend()[1] == 0).all())


def test_token_ranges_outside_the_rows_are_clamped():
    b = Batch([2, 3], [10, 20], 14, 2, 16, seed=10)
    b.q_start.copy_(torch.tensor([-7, 2, 1 << 30], dtype=torch.int32))
    b.attend()
    b.q_start.copy_(torch.tensor([5, 2, 0], dtype=torch.int32))
    out = b.attend()
    assert bool((out == 7).all())  # descending: nothing belongs to anyone
    assert ops.device_status() == 0


@pytest.mark.parametrize("new,cols", [([1] * 70, 300_000), ([200, 1, 57], 1_000_000)])
def test_tables_so_wide_that_the_split_takes_64_bits(new, cols):
    """The same bits as with a narrow table: only the host's bound on the work differs."""
    b = Batch(new, [37 * i % 613 for i in range(len(new))], 14, 2, 16, seed=16)
    want = b.attend()
    wide = torch.full((len(new), cols), -1, dtype=torch.int32, device="cuda")
    wide[:, :b.table.shape[1]] = b.table_dev
    b.table_dev = wide
    out = b.attend()
    assert torch.equal(out, want)
    b.check(out)


def test_many_heads_share_a_kv_head():
    """Up to 128 query heads per KV head: tiles of one token."""
    for H, KVH in ((128, 1), (34, 2), (100, 2)):
        b = Batch([1, 3, 40], [90, 5, 0], H, KVH, 16, seed=17)
        b.check(b.attend())


def test_calls_from_several_threads():
    import threading

    batches = [Batch([1] * 5, [300, 9, 77, 0, 1200], 14, 2, 16, seed=18), Batch([150, 2], [30, 500], 12, 12, 32, seed=19)]
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


def test_attention_graph_replays_with_other_lengths_and_pages():
    a = Batch([1, 1, 1, 1], [40, 3, 700, 0], 14, 2, 16, seed=11, extra_cols=30)
    b = Batch([1, 2, 0, 1], [900, 64, 5, 17], 14, 2, 16, seed=12, extra_cols=17)
    n = min(a.kp.shape[0], b.kp.shape[0])
    pool_k = torch.full((a.kp.shape[0] + b.kp.shape[0], 2, 16, 64), NAN, dtype=torch.bfloat16, device="cuda")
    pool_v = pool_k.clone()
    assert n > 0
    cols = max(a.table.shape[1], b.table.shape[1])
    table = torch.zeros((4, cols), dtype=torch.int32, device="cuda")
    q_start, kv_len = a.q_start.clone(), a.kv_len.clone()
    q = a.q.cuda()
    out = torch.zeros((4, 14 * 64), dtype=torch.bfloat16, device="cuda")
    run = lambda: ops.paged_attention(q, pool_k, pool_v, out, table, q_start, kv_len, 0.125)  # noqa: E731

    def load(x):
        pool_k[:x.kp.shape[0]].copy_(x.kp)
        pool_v[:x.vp.shape[0]].copy_(x.vp)
        table[:, :x.table.shape[1]].copy_(x.table_dev)
        q_start.copy_(x.q_start)
        kv_len.copy_(x.kv_len)
        q.copy_(x.q)

    load(a)
    run()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    out2 = torch.zeros_like(out)
    with torch.cuda.graph(g1):
        run()
    with torch.cuda.graph(g2):
        ops.paged_attention(q, pool_k, pool_v, out2, table, q_start, kv_len, 0.125)
    for x in (a, b, a):
        load(x)
        out.zero_()
        out2.zero_()
        torch.cuda.synchronize()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        for _ in range(5):  # both graphs at once: each has a workspace of its own
            with torch.cuda.stream(s1):
                g1.replay()
            with torch.cuda.stream(s2):
                g2.replay()
        torch.cuda.synchronize()
        x.check(out)
        assert torch.equal(out, out2)


def test_attention_on_two_streams_at_once():
    a = Batch([1] * 6, [5000, 90, 3000, 10, 400, 2], 14, 2, 16, seed=13)
    b = Batch([200, 1], [1000, 4000], 14, 2, 16, seed=14)
    want = a.attend(), b.attend()
    qa, qb = a.q.cuda(), b.q.cuda()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            ra = a.attend(qa)
        with torch.cuda.stream(s2):
            rb = b.attend(qb)
        got.append((ra, rb))
    torch.cuda.synchronize()
    for ra, rb in got:
        assert torch.equal(ra, want[0]) and torch.equal(rb, want[1])


def test_attention_agrees_with_the_contiguous_kernel():
    """Equal lengths: the paged result is the contiguous one within both kernels' rounding."""
    B, S, H, KVH, pos, page = 3, 90, 14, 2, 70, 16
    b = Batch([S] * B, [pos] * B, H, KVH, page, seed=15)
    k = torch.stack([x.transpose(0, 1) for x in b.k]).contiguous().cuda()
    v = torch.stack([x.transpose(0, 1) for x in b.v]).contiguous().cuda()
    q = b.q.view(B, S, H, 64).transpose(1, 2).contiguous().cuda()
    out = torch.empty((B, S, H * 64), dtype=torch.bfloat16, device="cuda")
    ops.attention(q, k, v, out, B, S, H, KVH, 64, pos, 0.125)
    got = b.attend()
    b.check(got)
    b.check(out.view(B * S, H * 64))


# ----------------------------------------------------------------------------- RoPE + page write


@pytest.mark.parametrize("D", [64, 16, 128])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("new,past,H,KVH,page", [([1], [0], 14, 2, 16), ([1] * 40, [i * 13 for i in range(40)], 14, 2, 16),
                                                 ([70, 0, 1, 129], [5, 9, 200, 0], 12, 12, 8),
                                                 ([3, 300], [47, 33], 9, 3, 48)])
def test_rope_kv_matches_oracle_bit_for_bit(D, rope, new, past, H, KVH, page):
    b = Batch(new, past, H, KVH, page, seed=20, pad=3, D=D)
    g = torch.Generator().manual_seed(21)
    qkv = torch.randn((b.T, (H + 2 * KVH) * D), generator=g).to(torch.bfloat16)
    top = max(x + y for x, y in zip(new, past))
    cos, sin = OQ.rope_tables(D, top, 1e6)
    wide = torch.zeros((b.T, (H + 2 * KVH) * D + 8), dtype=torch.bfloat16, device="cuda")
    wide[:, :-8] = qkv.cuda()
    q = torch.full((b.T, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
    want_k, want_v = b.kp.cpu().clone(), b.vp.cpu().clone()
    ops.paged_rope_kv(wide[:, :-8], cos.cuda() if rope else None, sin.cuda() if rope else None, q, b.kp, b.vp,
                      b.table_dev, b.q_start, b.kv_len)
    want_q = torch.full((b.T, H, D), 7.0, dtype=torch.bfloat16)
    for i, n in enumerate(new):
        if n == 0:
            continue
        t = b.starts[i]
        x = qkv[t:t + n].view(1, n, H + 2 * KVH, D).transpose(1, 2)
        turned = OQ.apply_rope(x[:, :H + KVH].contiguous(), cos, sin, past[i]) if rope else x[:, :H + KVH]
        want_q[t:t + n] = turned[0, :H].transpose(0, 1)
        for j in range(n):
            p = past[i] + j
            want_k[b.table[i, p // page], :, p % page] = turned[0, H:, j]
            want_v[b.table[i, p // page], :, p % page] = x[0, H + KVH:, j]
    assert torch.equal(q.cpu(), want_q)
    assert torch.equal(b.kp.cpu().view(torch.int16), want_k.view(torch.int16))  # bits: the poison too
    assert torch.equal(b.vp.cpu().view(torch.int16), want_v.view(torch.int16))
    assert ops.page_status() == 0


def test_rope_kv_equals_the_contiguous_kernel():
    B, S, H, KVH, pos = 2, 50, 14, 2, 13
    b = Batch([S] * B, [pos] * B, H, KVH, 16, seed=22)
    qkv = torch.randn((B * S, 18 * 64), generator=torch.Generator().manual_seed(23)).to(torch.bfloat16).cuda()
    cos, sin = (t.cuda() for t in OQ.rope_tables(64, 80, 1e6))
    q1 = torch.empty((B, H, S, 64), dtype=torch.bfloat16, device="cuda")
    kc, vc = (torch.zeros((B, KVH, 80, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.rope_kv(qkv, cos, sin, q1, kc, vc, B, S, H, KVH, 64, pos)
    q2 = torch.empty((B * S, H, 64), dtype=torch.bfloat16, device="cuda")
    ops.paged_rope_kv(qkv, cos, sin, q2, b.kp, b.vp, b.table_dev, b.q_start, b.kv_len)
    assert torch.equal(q2.view(B, S, H, 64).transpose(1, 2), q1)
    for i in range(B):
        pages = b.table_dev[i].long()
        for pool, cache in ((b.kp, kc), (b.vp, vc)):
            rows = pool[pages].transpose(1, 2).reshape(-1, KVH, 64)[pos:pos + S]
            assert torch.equal(rows, cache[i, :, pos:pos + S].transpose(0, 1))


def test_rope_kv_skips_what_has_no_place():
    """Missing pages, negative positions and positions past the tables: reported, nothing written elsewhere."""
    H, KVH = 14, 2
    b = Batch([2, 3, 1, 1], [10, -1, 40, 20], H, KVH, 16, seed=24)
    cos, sin = (t.cuda() for t in OQ.rope_tables(64, 32, 1e6))  # sequence 2 is past the tables
    b.table_dev[0, 0] = b.kp.shape[0]  # sequence 0 has no page
    before_k = b.kp.clone()
    qkv = torch.randn((b.T, 18 * 64), generator=torch.Generator().manual_seed(25)).to(torch.bfloat16).cuda()
    q = torch.full((b.T, H, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    assert ops.page_status() == 0
    ops.paged_rope_kv(qkv, cos, sin, q, b.kp, b.vp, b.table_dev, b.q_start, b.kv_len)
    assert ops.page_status() == 1 and ops.page_status() == 0
    left = (q == 7).all(-1).all(-1).tolist()
    assert left == [False, False, True, False, False, True, False]
    changed = (b.kp.view(torch.int16) != before_k.view(torch.int16)).any(-1).any(1).nonzero().tolist()
    where = sorted([[int(b.table[1, 0]), 0], [int(b.table[1, 0]), 1], [int(b.table[3, 1]), 4]])
    assert sorted(changed) == where


def test_rope_kv_with_starts_that_do_not_ascend():
    """Nothing outside the sequences' own pages is written, whatever the starts say."""
    b = Batch([3, 3, 3], [10, 20, 30], 14, 2, 16, seed=26)
    qkv = torch.randn((b.T, 18 * 64), generator=torch.Generator().manual_seed(27)).to(torch.bfloat16).cuda()
    for starts in ([0, 9, 3, 9], [9, 6, 3, 0], [0, 3, -2 ** 31, 9], [2 ** 31 - 1] * 4, [-5, 2, 40, 1]):
        b.q_start.copy_(torch.tensor(starts, dtype=torch.int64).to(torch.int32))
        b.kv_len.fill_(2 ** 31 - 1 if starts[0] == 0 else 12)
        kp, vp = b.kp.clone(), b.vp.clone()
        q = torch.full((b.T, 14, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.paged_rope_kv(qkv, None, None, q, kp, vp, b.table_dev, b.q_start, b.kv_len)
        used = {int(p) for p in b.table.flatten() if p >= 0}
        for pool, was in ((kp, b.kp), (vp, b.vp)):
            changed = (pool.view(torch.int16) != was.view(torch.int16)).flatten(1).any(1).nonzero().flatten().tolist()
            assert set(changed) <= used
    ops.page_status()


# ----------------------------------------------------------------------------- page copies


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int8])
@pytest.mark.parametrize("shape,n", [((3, 2, 40, 2, 16, 64), 1), ((3, 2, 40, 2, 16, 64), 17), ((1, 2, 1300, 1, 8, 64), 600),
                                     ((2, 2, 30, 5, 24, 16), 14), ((1, 1, 9, 1, 1, 16), 4)])
def test_copy_pages_matches_indexing(dtype, shape, n):
    g = torch.Generator().manual_seed(30)
    pool = torch.randint(-100, 100, shape, generator=g).to(dtype)
    perm = torch.randperm(shape[2], generator=g)
    dst = perm[:n]
    src = perm[n:][torch.randint(0, shape[2] - n, (n,), generator=g)]  # one page may go to several
    want = pool.clone()
    want[:, :, dst] = pool[:, :, src]
    got = pool.cuda()
    assert ops.copy_pages(got, src.tolist() if n < 5 else src, dst) is got
    assert torch.equal(got.cpu(), want)


def test_copy_pages_other_dimension_and_empty():
    pool = torch.arange(6 * 4 * 32, dtype=torch.float32).view(6, 4, 32).cuda()
    want = pool.clone()
    want[[0, 5]] = pool[[3, 3]]
    ops.copy_pages(pool, [3, 3], [0, 5], dim=0)
    assert torch.equal(pool, want)
    ops.copy_pages(pool, [], [], dim=0)
    ops.copy_pages(pool, torch.empty(0), torch.empty(0, dtype=torch.int64), dim=0)
    assert torch.equal(pool, want)


def test_copy_pages_in_a_graph():
    pool = torch.randn((2, 2, 20, 2, 16, 64), generator=torch.Generator().manual_seed(31)).to(torch.bfloat16).cuda()
    want = pool.clone()
    want[:, :, [1, 2]] = pool[:, :, [10, 11]]
    first = pool.clone()
    ops.copy_pages(pool, [10, 11], [1, 2])
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        ops.copy_pages(pool, [10, 11], [1, 2])
    pool.copy_(first)
    gr.replay()
    assert torch.equal(pool, want)


# ----------------------------------------------------------------------------- refusals that need a device


def test_refusals():
    b = Batch([1, 2], [4, 5], 14, 2, 16, seed=40)
    q, out = b.q.cuda(), torch.empty((3, 14 * 64), dtype=torch.bfloat16, device="cuda")
    args = [q, b.kp, b.vp, out, b.table_dev, b.q_start, b.kv_len, 0.125]

    def refused(exc, match, **swap):
        names = ["q", "k", "v", "out", "table", "q_start", "kv_len", "scale"]
        a = [swap.get(n, x) for n, x in zip(names, args)]
        with pytest.raises(exc, match=match):
            ops.paged_attention(*a)

    refused(TypeError, "int32", table=b.table_dev.long())
    refused(TypeError, "bf16", q=q.float())
    refused(ValueError, "rows", out=out[:2])
    refused(ValueError, "memory", out=q.view(3, 14 * 64))
    refused(ValueError, "batch", kv_len=b.kv_len[:1])
    refused(ValueError, "column", table=b.table_dev[:, :0])
    refused(ValueError, "rows of q must", q=q.transpose(1, 2).contiguous().transpose(1, 2))
    refused(RuntimeError, "scale", scale=0.0)
    refused(RuntimeError, "scale", scale=NAN)
    refused(RuntimeError, "multiple of 8", k=b.kp[:, :, :12].contiguous(), v=b.vp[:, :, :12].contiguous())
    refused(RuntimeError, "bad", q=q[:, :13].contiguous(), out=torch.empty((3, 13 * 64), dtype=torch.bfloat16,
                                                                                 device="cuda"))
    refused(ValueError, "CUDA", q=b.q)
    pool = torch.zeros((1, 2, 8, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    for src, dst, msg in (([0], [8], "outside"), ([-1], [2], "outside"), ([0, 1], [2, 2], "twice"), ([0, 1], [1, 3], "both"),
                          ([3], [3], "both"), ([0], [1, 2], "destinations"), ([2 ** 40], [1], "outside")):
        with pytest.raises((RuntimeError, ValueError), match=msg):
            ops.copy_pages(pool, src, dst)
    with pytest.raises(TypeError):
        ops.copy_pages(pool, torch.tensor([0]).cuda(), [1])
    with pytest.raises(TypeError):
        ops.copy_pages(pool, [0.5], [1])
    with pytest.raises(ValueError, match="contiguous"):
        ops.copy_pages(pool.transpose(2, 3), [0], [1])
    ops.copy_pages(pool, [0], [1])
    torch.cuda.synchronize()
