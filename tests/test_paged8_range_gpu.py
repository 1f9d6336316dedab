"""8-bit pages whose exponents lie far apart.  Tolerances as in test_paged8_gpu.py, with
what a result's rounding adds where it is tiny: bf16's numbers below 2^-126 are 2^-133
apart, so rounding to them is off by up to 2^-134, whatever the value; and with what
the least exponent adds to the loss of weights in fp16: there W = max p_k 2^e_k is that
of a vector of e = -80, whose largest code may be anything down to zero, so 2^-39 W
times a code of 448 is not bounded by the values themselves, but by 2^-39 2^-80 448 <
2^-110 a key.
"""

import math

import pytest
import torch
from test_paged8_gpu import DTYPES, Coded

from xb200 import ops

pytestmark = pytest.mark.gpu

# few rows with a CTA a unit, tiles of 32 keys, of 64 keys (8 and 16 rows each); many rows
VARIANTS = [([1] * 3, [90, 700, 300], 0), ([2] * 3, [90, 400, 300], 0), ([1] * 3, [90, 2100, 300], 0),
            ([2] * 3, [90, 2100, 300], 0), ([1] * 3, [90, 2100, 300], 3000), ([2] * 3, [90, 2100, 300], 3000),
            ([40, 1, 70], [90, 700, 300], 0)]


def _check(b, out, rows=slice(None)):
    o, a, lost = (x[rows] for x in b.exact())
    got = out.cpu().double().reshape(b.T, b.H, b.D)[rows]
    assert bool(torch.isfinite(got).all())
    tiny = 2.0 ** -134 + max(v.shape[0] for v in b.v) * 2.0 ** -110
    over = (got - o).abs() - (2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -12) * a + lost + tiny)
    assert float(over.max()) <= 0.0, (float(over.max()), int(over.argmax()))
    assert ops.device_status() == 0 and ops.page_status() == 0


def _shift(pool, held, table, positions, step, heads=slice(None)):
    """Values at some positions times 2^step, in the exponents and in what they stand for."""
    for p in positions:
        page, row = table[p // 16], p % 16
        pool[page, heads, row] += step if step > 0 else 256 + step
    at = torch.tensor(list(positions), dtype=torch.int64)
    held[at] = torch.ldexp(held[at], torch.tensor(step))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,past,cols", VARIANTS)
def test_scores_of_zero_between_large_factors(new, past, cols, dtype):
    """A query and keys that share no dimension, so large that their factors' product is no fp32 number."""
    b = Coded(dtype, new, past, 14, 2, 16, seed=90, extra_cols=cols)
    b.kp.view(torch.uint8)[..., 0] = 0
    for i, k in enumerate(b.k):
        k[..., 0] = 0
        _shift(b.ks, k, b.table[i], range(k.shape[0]), 94)
    b.q.zero_()
    b.q[..., 0] = 2.0 ** 60
    b.check(b.attend())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,past,cols", VARIANTS[:-1])  # of many rows the scores stay below 2^30
@pytest.mark.parametrize("up,down", [(118, -70), (118, 2), (-118, 94), (126, -60)])
def test_huge_queries_and_small_keys(up, down, new, past, cols, dtype):
    """Products of queries and codes that are no fp32 numbers, of scores that are: one key has all the weight."""
    b = Coded(dtype, new, past, 14, 2, 16, seed=91, extra_cols=cols)
    for i, k in enumerate(b.k):
        _shift(b.ks, k, b.table[i], range(k.shape[0]), down)
    size = b.q.float().abs().amax(-1, keepdim=True).log2().ceil()  # every row's largest below 2^up
    b.q = torch.ldexp(b.q.float(), up - size).to(torch.bfloat16)
    b.check(b.attend())


def _zero(b, i, positions):
    """Values of zeros, as the write leaves them."""
    for p in positions:
        page, row = b.table[i, p // 16], p % 16
        b.vp.view(torch.uint8)[page, :, row], b.vs[page, :, row] = 0, 47
        b.v[i][p] = 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("step", [53, 60, 67, 80, 100, 112])
def test_a_key_of_zeros_beside_one_of_large_values(step, dtype):
    """Two keys alike: half of the second one's value."""
    b = Coded(dtype, [1], [1], 14, 2, 16, seed=92)
    b.kp.view(torch.uint8)[...] = 0
    b.k[0].zero_()
    _zero(b, 0, [0])
    _shift(b.vs, b.v[0], b.table[0], [1], step)
    out = b.attend()
    _check(b, out)
    want = (b.v[0][1] / 2).repeat_interleave(7, 0).reshape(1, -1)
    assert bool(((out.cpu().double() - want).abs() <= want.abs() * 2.0 ** -8).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,past,cols", VARIANTS)
@pytest.mark.parametrize("which", ["first half", "second half", "every second", "all but one", "one", "runs"])
@pytest.mark.parametrize("step", [60, 100, -60])
def test_keys_of_zeros_among_values_of_any_size(step, which, new, past, cols, dtype):
    """In one tile, in tiles one after the other, in parts of different warps and CTAs."""
    b = Coded(dtype, new, past, 14, 2, 16, seed=93, extra_cols=cols)
    for i, v in enumerate(b.v):
        n = v.shape[0]
        zeros = {"first half": range(n // 2), "second half": range(n // 2, n), "every second": range(0, n, 2),
                 "all but one": [p for p in range(n) if p != n // 3], "one": [n // 2],
                 "runs": [p for p in range(n) if p // 32 % 3 == 1]}[which]
        _zero(b, i, zeros)
        _shift(b.vs, v, b.table[i], sorted(set(range(n)) - set(zeros)), step)
    _check(b, b.attend())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,past,cols", VARIANTS)
def test_values_of_all_sizes_at_once(new, past, cols, dtype):
    """Exponents of -80 to 110, in steps that change from position to position and from run to run."""
    b = Coded(dtype, new, past, 14, 2, 16, seed=94, extra_cols=cols)
    for i, v in enumerate(b.v):
        for step, at in ((110, 0), (55, 1), (-60, 3), (-30, 4), (85, 40), (-50, 41)):
            _shift(b.vs, v, b.table[i], [p for p in range(v.shape[0]) if (p % 5 == at if at < 5 else p % 5 == 2 and
                                                                          p // 100 % 2 == at - 40)], step)
    _check(b, b.attend())


def _determined(b, limit):
    """Rows [T, H] whose result fp32 scores settle: all but those in which some other key's score is so close to the
    largest that the sums' rounding decides.  The 64 products of a score are exact, their sum is off by at most 2^-23 of A =
    sum |q k| an addition (a tensor core cuts off), so two scores by 64 x 2 x 2^-23 A = 2^-16 A, and where they are 40
    further apart than that the other weights are lost below 2^-40.  Scores have to stay below `limit`."""
    ok = torch.zeros((b.T, b.H), dtype=torch.bool)
    for i, n in enumerate(b.new):
        t, L = b.starts[i], b.k[i].shape[0]
        k = b.k[i].double().repeat_interleave(b.H // b.KVH, 1).transpose(0, 1)  # [H, L, D]
        q = b.q[t:t + n].double().transpose(0, 1) * (0.125 / math.log(2.0))
        hidden = torch.arange(L)[None, :] > L - n + torch.arange(n)[:, None]
        s, a = ((x @ y.transpose(1, 2)).masked_fill(hidden, -math.inf) for x, y in ((q, k), (q.abs(), k.abs())))
        top = s.topk(min(2, L), -1).values
        gap = top[..., 0] - top[..., -1] if L > 1 else torch.full((b.H, n), math.inf, dtype=torch.float64)
        one = (torch.isfinite(s).sum(-1) == 1) | (gap > 2.0 ** -16 * a.amax(-1) + 40)
        ok[t:t + n] = (one & (s.masked_fill(hidden, 0).abs().amax(-1) < limit)).t()
    return ok


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,past,cols", VARIANTS)
@pytest.mark.parametrize("step", range(17, 25))
def test_scores_whose_neighbours_are_more_than_one_apart(step, new, past, cols, dtype):
    """Scores of 2^22 to 2^30: fp32 there has steps of 0.5 to 128, and fp16 ends at 2^16."""
    b = Coded(dtype, new, past, 14, 2, 16, seed=95, extra_cols=cols)
    b.q = torch.ldexp(b.q.float(), torch.tensor(step)).to(torch.bfloat16)
    ok = _determined(b, math.inf if max(new) < 3 else 2.0 ** 30)
    assert step > 21 or ok.float().mean() > 0.9
    _check(b, b.attend(), ok)
