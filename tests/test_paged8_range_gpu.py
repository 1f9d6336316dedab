"""8-bit pages whose exponents lie far apart.  Tolerances as in test_paged8_gpu.py."""

import pytest
import torch
from test_paged8_gpu import DTYPES, Coded

pytestmark = pytest.mark.gpu

# few rows with a CTA a unit, tiles of 32 keys, of 64 keys (8 and 16 rows each); many rows
VARIANTS = [([1] * 3, [90, 700, 300], 0), ([2] * 3, [90, 400, 300], 0), ([1] * 3, [90, 2100, 300], 0),
            ([2] * 3, [90, 2100, 300], 0), ([1] * 3, [90, 2100, 300], 3000), ([2] * 3, [90, 2100, 300], 3000),
            ([40, 1, 70], [90, 700, 300], 0)]


def _shift(pool, held, table, positions, step, heads=slice(None)):
    """Values at some positions times 2^step, in the exponents and in what they stand for."""
    for p in positions:
        page, row = table[p // 16], p % 16
        pool[page, heads, row] += step if step > 0 else 256 + step
    at = torch.as_tensor(positions)
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
