"""8-bit pages of the paged KV cache: write, reading back and attention.

What codes stand for is a bf16 number, so reading back is exact, and the attention
is held to the 64-bit attention over those numbers with the tolerance of the bf16
kernels (test_paged_gpu.py): the weights are rounded to no fewer bits, the codes
not at all.  But codes are often exactly zero where others of the same vector are not, so an
element may be the sum of tiny weights alone, for which the ranges of the
weights' types count.  A weight p_k, in fp32 relative to the largest, vanishes
below 2^-126: L keys are off by L 2^-126 max |v| at most.  In fp16 it is 2^14 p_k
2^e_k / W, with e_k the exponent of value k and W = max p_k 2^e_k; where that is
below fp16's normal numbers its rounding is off by 2^-25, 2^-39 W in all, times a
code of at most 448 <= 2 max_d |v_kd| / 2^e_k: L keys are off by L 2^-38 max_k (p_k
max_d |v_kd|).  Both are added.  Rows that no sequence uses and rows behind a sequence's last
position hold codes of NaN (e4m3) or -128 (int8) and the exponent byte 255.
"""

import math

import pytest
import torch
from test_paged_gpu import SHAPES, Batch

from oracle import qwen as OQ
from xb200 import ops

pytestmark = pytest.mark.gpu

NAN = float("nan")
DTYPES = [torch.int8, torch.float8_e4m3fn]
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LAST = {torch.int8: 248, torch.float8_e4m3fn: 246}


def quantise(x, dtype):
    """Codes and exponent bytes of bf16 vectors on the host: the definition, exponent by exponent."""
    x = x.double()
    top = x.abs().amax(-1)
    most = LAST[dtype] - 127
    e = torch.full(top.shape, most, dtype=torch.int64)
    for k in range(most - 1, -81, -1):
        e = torch.where(top <= MOST[dtype] * 2.0 ** k, k, e)  # the smallest that holds it
    bad = ~x.isfinite().all(-1)
    y = torch.ldexp(torch.where(bad[..., None], 0.0, x), -e[..., None]).clamp(-MOST[dtype], MOST[dtype])
    codes = (y.round() if dtype is torch.int8 else y.float()).to(dtype)  # y has 8 bits: the step through fp32 is exact
    return codes, torch.where(bad, 255, e + 127).to(torch.uint8)


def values(codes, byte):
    """What they stand for, in 64 bits."""
    x = torch.ldexp(codes.double(), (byte.long() - 127)[..., None])
    return torch.where((byte == 255)[..., None], NAN, x)


class Coded(Batch):
    """A ragged batch whose pool is quantised; k and v become what the codes stand for."""

    def __init__(self, dtype, *a, **kw):
        layout = kw.pop("layout", "nhpd")
        super().__init__(*a, **kw)
        self.dtype = dtype
        g = torch.Generator().manual_seed(99)
        n, KVH, P, D = self.kp.shape
        pools = []
        for held in (self.k, self.v):
            codes = torch.full((n, KVH, P, D), 0x7F if dtype is not torch.int8 else -128, dtype=torch.int8).view(dtype)
            byte = torch.full((n, KVH, P), 255, dtype=torch.uint8)
            for b, x in enumerate(held):
                size = torch.exp(torch.randn(x.shape[:2], generator=g))[..., None]
                c, e = quantise((x.float() * size).to(torch.bfloat16), dtype)
                held[b] = values(c, e)
                for p in range(x.shape[0]):
                    i, r = self.table[b, p // P], p % P
                    codes[i, :, r], byte[i, :, r] = c[p], e[p]
            pools.append((codes.cuda(), byte.cuda()))
        (self.kp, self.ks), (self.vp, self.vs) = pools
        if layout == "joint":  # K and V, codes and exponents, side by side
            both, ex = torch.stack([self.kp, self.vp], 1), torch.stack([self.ks, self.vs], 1)
            self.kp, self.vp, self.ks, self.vs = both[:, 0], both[:, 1], ex[:, 0], ex[:, 1]
        elif layout == "rows":  # heads inside rows; exponents of a wider tensor
            self.kp, self.vp = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (self.kp, self.vp))
            wide = torch.zeros((n, KVH, P + 8), dtype=torch.uint8, device="cuda")
            wide[..., :P] = self.ks
            self.ks = wide[..., :P]

    def attend(self, q=None, out=None, scale=0.125):
        q = self.q.cuda() if q is None else q
        if out is None:
            out = torch.full((self.T, self.H * self.D), 7.0, dtype=torch.bfloat16, device="cuda")
        return ops.paged_attention(q, self.kp, self.vp, out, self.table_dev, self.q_start, self.kv_len, scale, self.ks,
                                   self.vs)

    def exact(self, scale=0.125):
        """(o, sum of p |v|, what the weights' ranges may lose) in 64 bits."""
        o, a = super().exact(scale)
        lost = torch.zeros((self.T, self.H, 1), dtype=torch.float64)
        rep = self.H // self.KVH
        for b, n in enumerate(self.new):
            t, L = self.starts[b], self.k[b].shape[0]
            if n == 0 or L == 0:
                continue
            k = self.k[b].double().repeat_interleave(rep, 1).transpose(0, 1)  # [H, L, D]
            top = self.v[b].double().abs().amax(-1).repeat_interleave(rep, 1).t()[:, None]  # [H, 1, L]
            pos = L - n + torch.arange(n)
            s = self.q[t:t + n].double().transpose(0, 1) @ k.transpose(1, 2) * scale
            s = s.masked_fill(torch.arange(L)[None, :] > pos[:, None], -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1))
            x = L * (2.0 ** -38 * (p * top).amax(-1) + 2.0 ** -126 * top.amax(-1))
            lost[t:t + n, :, 0] = x.t()
        return o, a, lost

    def check(self, out, scale=0.125):
        o, a, lost = self.exact(scale)
        got = out.cpu().double().reshape(self.T, self.H, self.D)
        assert bool(torch.isfinite(got).all())
        over = (got - o).abs() - (2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -12) * a + lost)
        assert float(over.max()) <= 0.0, (float(over.max()), int(over.argmax()))
        assert ops.device_status() == 0 and ops.page_status() == 0


# ----------------------------------------------------------------------------- attention


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_matches_64_bits(case, dtype):
    new, past, H, KVH, page = SHAPES[case]
    b = Coded(dtype, new, past, H, KVH, page, seed=case)
    out = b.attend()
    b.check(out)
    assert torch.equal(out, b.attend())  # joined in a fixed order


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["joint", "rows"])
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 1, 200]])
def test_attention_over_strided_pages_and_pitched_rows(layout, new, dtype):
    b = Coded(dtype, new, [40, 513, 3], 14, 2, 16, seed=3, layout=layout, extra_cols=5)
    wide = torch.zeros((b.T, 18 * 64), dtype=torch.bfloat16, device="cuda")
    q = wide[:, :14 * 64].view(b.T, 14, 64)
    q.copy_(b.q)
    wide_out = torch.full((b.T, 16 * 64), 7.0, dtype=torch.bfloat16, device="cuda")
    b.attend(q, wide_out[:, 64:15 * 64])
    b.check(wide_out[:, 64:15 * 64])
    assert bool((wide_out[:, :64] == 7).all()) and bool((wide_out[:, 15 * 64:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,past", [([4, 1], [-2, 10]), ([1, 2], [-1, -2]), ([150, 20], [-140, 5])])
def test_tokens_without_a_key_get_zeros(new, past, dtype):
    b = Coded(dtype, new, past, 14, 2, 16, seed=5, pad=3)
    out = b.attend()
    b.check(out)
    assert bool((out[:-past[0]] == 0).all()) and bool((out[-3:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1, 1], [60, 1, 90]])
def test_bad_pages_read_as_zeros_and_are_reported(new, dtype):
    b = Coded(dtype, new, [100, 50, 200], 14, 2, 16, seed=8)
    assert ops.page_status() == 0
    for j, bad in ((0, -1), (2, b.kp.shape[0]), (3, 2 ** 31 - 1), (4, -2 ** 31)):
        b.table_dev[2, j] = bad
        b.k[2][j * 16:j * 16 + 16] = 0
        b.v[2][j * 16:j * 16 + 16] = 0
    out = b.attend()
    assert ops.page_status() == 1
    b.check(out)  # the flag is clear again


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 1, 33, 64]])
def test_sequences_that_share_pages(new, dtype):
    """Four sequences name the same pages of an earlier part, one of them a page twice."""
    b = Coded(dtype, new, [64] * 4, 12, 12, 16, seed=9, extra_cols=200)  # a table larger than the pool
    for i in range(1, 4):
        b.table_dev[i, :4] = b.table_dev[0, :4]
        for x in (b.k, b.v):
            x[i][:64] = x[0][:64]
    b.table_dev[3, 1] = b.table_dev[3, 0]
    for x in (b.k, b.v):
        x[3][16:32] = x[3][:16]
    b.check(b.attend())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1] * 3, [30, 70, 1]])
@pytest.mark.parametrize("ratio", [1e-20, 1e-9, 1e9, 1e20])
def test_values_and_keys_of_very_different_sizes(ratio, new, dtype):
    """Half of the values are `ratio` times the others, the queries and keys of one head far larger and smaller."""
    b = Coded(dtype, new, [90, 200, 31], 14, 2, 16, seed=12)
    step = round(math.log2(ratio))
    for i in range(3):
        for p in range(0, b.v[i].shape[0], 2):
            page, row = b.table[i, p // 16], p % 16
            b.vs[page, :, row] += step if step > 0 else 256 + step
            b.v[i][p] = torch.ldexp(b.v[i][p], torch.tensor(step))
        for p in range(b.k[i].shape[0]):
            page, row = b.table[i, p // 16], p % 16
            b.ks[page, 1, row] += 40
            b.k[i][p, 1] = torch.ldexp(b.k[i][p, 1], torch.tensor(40))
    b.q[:, 7:] = torch.ldexp(b.q[:, 7:].float(), torch.tensor(-40)).to(torch.bfloat16)
    b.check(b.attend())


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_stays_with_the_tokens_that_see_it(dtype):
    b = Coded(dtype, [40, 1], [0, 30], 14, 2, 16, seed=6)
    clean = b.attend().view(b.T, 14, 64)
    b.q[3, 5, 0] = NAN
    out = b.attend().view(b.T, 14, 64)
    hit = torch.isnan(out).any(-1)
    assert hit.nonzero().tolist() == [[3, 5]] and torch.equal(out[~hit], clean[~hit])
    b.q = torch.nan_to_num(b.q)
    for pool, scale in ((b.kp, b.ks), (b.vp, b.vs)):
        page, row = int(b.table[1, 1]), 4  # position 20 of sequence 1
        was = pool[page, 0, row].clone(), scale[page, 0, row].clone()
        pool[page, 0, row], scale[page, 0, row] = 0, 255  # as the write leaves a vector with a NaN
        bad = torch.isnan(b.attend().view(b.T, 2, 7 * 64)).any(-1).cpu()
        assert bad[:, 0].tolist() == [False] * 40 + [True] and not bool(bad[:, 1].any())
        pool[page, 0, row], scale[page, 0, row] = was


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [50, 2, 0, 90]])
def test_graph_replays_with_other_lengths_and_on_two_streams(new, dtype):
    b = Coded(dtype, new, [40, 3, 700, 0], 14, 2, 16, seed=11, extra_cols=9)
    want = b.attend()
    q = b.q.cuda()
    short = torch.minimum(b.kv_len, torch.tensor([30, 2, 300, 1], dtype=torch.int32, device="cuda").clamp(
        min=b.q_start.diff().max().item() if max(new) == 1 else 0))
    full = b.kv_len.clone()
    b.kv_len.copy_(short)
    other = b.attend()
    outs, graphs = [torch.zeros_like(want) for _ in range(2)], []
    for out in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.attend(q, out)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for lens, expect in ((full, want), (short, other), (full, want)):
        b.kv_len.copy_(lens)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        rows = slice(0, sum(new))
        assert all(torch.equal(o[rows], expect[rows]) for o in outs)


# ----------------------------------------------------------------------------- write


def _write(b, qkv, cos, sin, H, D):
    q = torch.full((b.T, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_rope_kv(qkv, cos, sin, q, b.kp, b.vp, b.table_dev, b.q_start, b.kv_len, b.ks, b.vs)
    return q


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 16, 128, 512])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("new,past,H,KVH,page", [([1], [0], 14, 2, 16), ([1] * 40, [i * 13 for i in range(40)], 14, 2, 16),
                                                 ([70, 0, 1, 129], [5, 9, 200, 0], 12, 12, 8),
                                                 ([3, 30], [47, 33], 9, 3, 48),
                                                 ([2001, 0, 1, 1, 0, 1700], [3, 2, 40, 0, 9, 16], 3, 1, 16)])
def test_write_quantises_what_a_bf16_page_would_hold(D, rope, new, past, H, KVH, page, dtype):
    """Few tokens have a warp each, more than a GPU's 3552 warps half of one (up to D = 256)."""
    b = Coded(dtype, new, past, H, KVH, page, seed=20, pad=3, D=D)
    plain = Batch(new, past, H, KVH, page, seed=20, pad=3, D=D)
    g = torch.Generator().manual_seed(21)
    qkv = (torch.randn((b.T, (H + 2 * KVH) * D), generator=g) * torch.exp(2 * torch.randn((b.T, 1), generator=g)))
    qkv = qkv.to(torch.bfloat16).cuda()
    top = max(x + y for x, y in zip(new, past))
    cos, sin = (t.cuda() for t in OQ.rope_tables(D, top, 1e6)) if rope else (None, None)
    want = [x.cpu().clone() for x in (b.kp, b.vp, b.ks, b.vs)]
    q = _write(b, qkv, cos, sin, H, D)
    want_q = torch.full_like(q, 7.0)
    ops.paged_rope_kv(qkv, cos, sin, want_q, plain.kp, plain.vp, plain.table_dev, plain.q_start, plain.kv_len)
    assert torch.equal(q, want_q)
    for pool, codes, byte in ((plain.kp.cpu(), want[0], want[2]), (plain.vp.cpu(), want[1], want[3])):
        seq = torch.tensor([i for i, n in enumerate(new) for _ in range(n)])
        p = torch.tensor([past[i] + j for i, n in enumerate(new) for j in range(n)])
        at = b.table[seq, p // page].long(), slice(None), p % page
        codes.view(torch.uint8)[at], byte[at] = (x.view(torch.uint8) for x in quantise(pool[at], dtype))
    for got, expect in zip((b.kp, b.vp, b.ks, b.vs), want):  # bits: what was there before too
        assert torch.equal(got.cpu().view(torch.uint8), expect.view(torch.uint8))
    assert ops.page_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_at_the_borders_of_the_codes(dtype):
    """Vectors of zeros, of the largest and smallest numbers, at ties, around a change of exponent, with infinities and NaN."""
    M, big = MOST[dtype], torch.finfo(torch.bfloat16).max
    ramp = torch.arange(64.0)
    rows = [torch.zeros(64), -torch.zeros(64), torch.full((64,), big), torch.full((64,), -big), ramp * (big / 64),
            torch.full((64,), 2.0 ** -130), ramp * 2.0 ** -86, ramp * 2.0 ** -133, ramp - 0.5, 127 - ramp / 2,
            ramp * 0.5 - 16, 2.0 ** ramp.sub(40), 2.0 ** (ramp / 8 - 4), (ramp - 32) / 64]
    for m in (M, M * (1 + 2 ** -7), M * (1 - 2 ** -8), -M, 1.0, 255.0, 2.0 ** 100 * M, 2.0 ** -70 * M):
        rows.append(torch.cat([torch.tensor([m]), (ramp[1:] + 0.5) * (m / 130)]))
    for bad in (math.inf, -math.inf, NAN):
        r = torch.randn(64, generator=torch.Generator().manual_seed(1))
        r[17] = bad
        rows.append(r)
    k = torch.stack(rows).to(torch.bfloat16)
    T = k.shape[0]
    b = Coded(dtype, [T], [0], 1, 1, 16, seed=30)
    qkv = torch.cat([torch.zeros_like(k), k, k.flip(0)], 1).cuda()
    _write(b, qkv, None, None, 1, 64)
    k_out, v_out = (torch.empty((T, 1, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.paged_read_kv(k_out, v_out, b.kp, b.vp, b.table_dev, b.q_start, b.kv_len, b.ks, b.vs)
    codes, byte = quantise(k, dtype)
    pages, row = b.table[0, torch.arange(T) // 16].long(), torch.arange(T) % 16
    assert torch.equal(b.ks.cpu()[pages, 0, row], byte)
    assert torch.equal(b.kp.cpu()[pages, 0, row].view(torch.uint8), codes.view(torch.uint8))
    assert torch.equal(b.vp.cpu()[pages, 0, row].view(torch.uint8), codes.flip(0).view(torch.uint8))
    want = values(codes, byte)
    assert torch.equal(torch.nan_to_num(k_out.cpu()[:, 0].double(), 5.0), torch.nan_to_num(want, 5.0))
    assert torch.equal(torch.isnan(k_out.cpu()[:, 0]), torch.isnan(want))
    # half a step at most, but where exponents end
    ok = (byte > 47) & (byte < LAST[dtype])
    x, y = k[ok].double(), want[ok]
    step = torch.exp2(byte[ok].double() - 127)[:, None]
    half = step / 2 if dtype is torch.int8 else torch.maximum(x.abs() * 2.0 ** -4, step * 2.0 ** -10)
    assert bool(((x - y).abs() <= half).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_skips_what_has_no_place(dtype):
    H = 14
    b = Coded(dtype, [2, 3, 1, 1], [10, -1, 40, 20], H, 2, 16, seed=24)
    cos, sin = (t.cuda() for t in OQ.rope_tables(64, 32, 1e6))  # sequence 2 is past the tables
    b.table_dev[0, 0] = b.kp.shape[0]  # sequence 0 has no page
    was_k, was_s = b.kp.clone(), b.vs.clone()
    qkv = torch.randn((b.T, 18 * 64), generator=torch.Generator().manual_seed(25)).mul(100).to(torch.bfloat16).cuda()
    assert ops.page_status() == 0
    q = _write(b, qkv, cos, sin, H, 64)
    assert ops.page_status() == 1 and ops.page_status() == 0
    assert (q == 7).all(-1).all(-1).tolist() == [False, False, True, False, False, True, False]
    where = sorted([[int(b.table[1, 0]), 0], [int(b.table[1, 0]), 1], [int(b.table[3, 1]), 4]])
    changed = (b.kp.view(torch.uint8) != was_k.view(torch.uint8)).any(-1).any(1).nonzero().tolist()
    assert sorted(changed) == where
    assert sorted((b.vs != was_s).any(1).nonzero().tolist()) == where


# ----------------------------------------------------------------------------- reading back


@pytest.mark.parametrize("dtype", [torch.bfloat16, *DTYPES])
@pytest.mark.parametrize("D", [64, 16, 8, 24])
@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("new,past,H,KVH,page", [([1], [0], 14, 2, 16), ([2, 0, 5], [30, 9, 300], 12, 12, 8),
                                                 ([1] * 70, [i * 7 for i in range(70)], 9, 3, 48)])
def test_read_returns_what_the_pages_hold(new, past, H, KVH, page, whole, D, dtype):
    if dtype is not torch.bfloat16 and D % 16:
        pytest.skip("8-bit rows are multiples of 16")
    b = Batch(new, past, H, KVH, page, seed=40, D=D) if dtype is torch.bfloat16 else Coded(dtype, new, past, H, KVH, page,
                                                                                           seed=40, D=D)
    counts = [x.shape[0] for x in b.k] if whole else new
    starts = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()
    T = sum(counts)
    wide = torch.full((T + 2, KVH * D + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    k_out = torch.full((T + 2, KVH, D), 7.0, dtype=torch.bfloat16, device="cuda")
    v_out = wide[:, 8:8 + KVH * D]
    scales = () if dtype is torch.bfloat16 else (b.ks, b.vs)
    got = ops.paged_read_kv(k_out, v_out, b.kp, b.vp, b.table_dev, starts, b.kv_len, *scales)
    assert got[0] is k_out and got[1] is v_out
    for held, out in ((b.k, k_out), (b.v, v_out.view(T + 2, KVH, D))):
        want = torch.cat([x[x.shape[0] - n:] for x, n in zip(held, counts)])
        assert torch.equal(out[:T].cpu().double(), want.double())
        assert bool((out[T:] == 7).all())
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + KVH * D:] == 7).all())
    assert ops.page_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, *DTYPES])
def test_read_of_missing_pages_gives_zeros(dtype):
    b = Batch([2, 3], [10, -1], 14, 2, 16, seed=41) if dtype is torch.bfloat16 else Coded(dtype, [2, 3], [10, -1], 14, 2,
                                                                                          16, seed=41)
    b.table_dev[0, 0] = -1
    k_out, v_out = (torch.full((5, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    scales = () if dtype is torch.bfloat16 else (b.ks, b.vs)
    ops.paged_read_kv(k_out, v_out, b.kp, b.vp, b.table_dev, b.q_start, b.kv_len, *scales)
    assert ops.page_status() == 1 and ops.page_status() == 0
    assert bool((k_out[:3] == 0).all()) and bool((v_out[:3] == 0).all())  # no page, no page, no position
    assert torch.equal(k_out[3:].cpu().double(), b.k[1].double())
    b.q_start.copy_(torch.tensor([5, 2, 0], dtype=torch.int32))
    k_out.fill_(7)
    ops.paged_read_kv(k_out, v_out, b.kp, b.vp, b.table_dev, b.q_start, b.kv_len, *scales)
    assert bool((k_out == 7).all())
    ops.page_status()


# ----------------------------------------------------------------------------- refusals that need a device


def test_refusals():
    b = Coded(torch.int8, [1, 2], [4, 5], 14, 2, 16, seed=50)
    q, out = b.q.cuda(), torch.empty((3, 14 * 64), dtype=torch.bfloat16, device="cuda")
    names = ["q", "k", "v", "out", "table", "q_start", "kv_len", "scale", "ks", "vs"]
    args = [q, b.kp, b.vp, out, b.table_dev, b.q_start, b.kv_len, 0.125, b.ks, b.vs]

    def refused(exc, match, **swap):
        with pytest.raises(exc, match=match):
            ops.paged_attention(*[swap.get(n, x) for n, x in zip(names, args)])

    refused(ValueError, "k_scale", ks=None)
    refused(ValueError, "k_scale", vs=None)
    refused(ValueError, "k_scale", k=b.kp.to(torch.bfloat16), v=b.vp.to(torch.bfloat16))
    refused(TypeError, "both", k=b.kp.view(torch.float8_e4m3fn))
    refused(TypeError, "both", k=b.kp.view(torch.uint8), v=b.vp.view(torch.uint8))
    refused(TypeError, "both", k=b.kp.view(torch.float8_e5m2), v=b.vp.view(torch.float8_e5m2))
    refused(ValueError, "uint8", ks=b.ks[:, :1])
    refused(ValueError, "uint8", vs=b.vs.view(torch.int8))
    refused(ValueError, "contiguous", ks=b.ks.transpose(1, 2).contiguous().transpose(1, 2))
    refused(RuntimeError, "multiples of 8", ks=torch.zeros((b.ks.shape[0], 2, 20), dtype=torch.uint8,
                                                          device="cuda")[:, :, :16])
    refused(ValueError, "CUDA", ks=b.ks.cpu())
    refused(RuntimeError, "8-byte", ks=torch.zeros(b.ks.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(b.ks.shape))
    refused(RuntimeError, "scale", scale=-1.0)
    narrow = torch.zeros((b.kp.shape[0], 2, 16, 72), dtype=torch.int8, device="cuda")[..., :64]
    refused(RuntimeError, "multiples of 16", k=narrow)
    k_out = torch.empty((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="memory"):
        ops.paged_read_kv(k_out, k_out, b.kp, b.vp, b.table_dev, b.q_start, b.kv_len, b.ks, b.vs)
    with pytest.raises(ValueError, match="rows"):
        ops.paged_read_kv(k_out, k_out[:2].clone(), b.kp, b.vp, b.table_dev, b.q_start, b.kv_len, b.ks, b.vs)
    with pytest.raises(TypeError, match="bf16"):
        ops.paged_read_kv(k_out.float(), k_out, b.kp, b.vp, b.table_dev, b.q_start, b.kv_len, b.ks, b.vs)
    empty = k_out[:0]
    ops.paged_read_kv(empty, empty.clone(), b.kp, b.vp, b.table_dev, b.q_start, b.kv_len, b.ks, b.vs)
    torch.cuda.synchronize()
    assert ops.page_status() == 0
