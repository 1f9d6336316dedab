"""The selection of beam search against its definition in 64 bits.

Tolerance of the sums: they are formed in 64 bits and rounded to fp32 once
(2^-24 of the value), but for the log-sum: each exponential is off by at most
2^-22 (its own error) + 2^-24 |x - max| (its argument's two roundings, times ln 2
and log2 e) and the fp32 sums of at most 2^14 terms a thread by 2^-24 an addition
in the worst case, far less at random: 2^-17 absolute in all.
Sums that the definition has closer together than that may change places.
"""

import math

import pytest
import torch

from xb200 import ops

pytestmark = pytest.mark.gpu

INF = math.inf
OFF = 2.0 ** -17


def exact(logits, scores, count):
    G, K = scores.shape
    V = logits.shape[1]
    x = logits.cpu().double()
    total = scores.cpu().double().reshape(-1, 1) + x - torch.logsumexp(x, 1, keepdim=True)
    total = torch.where(total.isfinite(), total, -INF).view(G, K * V)
    best, at = total.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :count], at[:, :count]
    if best.shape[1] < count:
        best = torch.nn.functional.pad(best, (0, count - best.shape[1]), value=-INF)
        at = torch.nn.functional.pad(at, (0, count - at.shape[1]))
    none = best == -INF
    return best, (at // V).masked_fill(none, -1), (at % V).masked_fill(none, -1), total.view(G, K, V)


def check(logits, scores, count, exactly=True):
    values, parents, tokens = ops.beam_select(logits, scores, count)
    best, p, t, total = exact(logits, scores, count)
    G = scores.shape[0]
    assert values.shape == parents.shape == tokens.shape == (G, count)
    assert values.dtype is torch.float32 and parents.dtype is tokens.dtype is torch.int64
    values, parents, tokens = values.cpu().double(), parents.cpu(), tokens.cpu()
    none = best == -INF
    assert torch.equal(values == -INF, none)
    assert bool((parents[none] == -1).all()) and bool((tokens[none] == -1).all())
    err = (values - best).masked_fill(none, 0).abs()
    assert bool((err <= OFF + 2.0 ** -24 * best.masked_fill(none, 0).abs()).all()), float(err.max())
    if exactly:
        assert torch.equal(parents, p) and torch.equal(tokens, t)
    else:  # near ties may change places: what was chosen has the sum it claims, and nothing twice
        g = torch.arange(G)[:, None].expand_as(p)
        own = total[g, parents.clamp(min=0), tokens.clamp(min=0)]
        assert bool(((own - best).masked_fill(none, 0).abs() <= 2 * OFF).all())
        for i in range(G):
            pairs = [(a, b) for a, b in zip(parents[i].tolist(), tokens[i].tolist()) if a >= 0]
            assert len(set(pairs)) == len(pairs)
    return values, parents, tokens


def make(G, K, V, dtype=torch.float32, seed=0, pitch=0, offset=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((G * K, V), generator=g) * 3
    flat = torch.full((offset + G * K * (V + pitch),), float("nan"), dtype=dtype, device="cuda")
    rows = flat[offset:].view(G * K, V + pitch)[:, :V]
    rows.copy_(x)
    scores = (torch.randn((G, K), generator=g) * 2 - 20).cuda()
    return rows, scores


SIZES = [  # G, K, V, count
    (1, 1, 1, 1), (1, 1, 1, 8), (2, 3, 2, 6), (1, 4, 7, 8), (3, 2, 31, 4), (1, 4, 1000, 8), (5, 5, 4097, 10),
    (1, 4, 50257, 8), (2, 16, 50257, 32), (1, 64, 300, 64), (1, 33, 8192, 64), (70, 2, 2049, 4), (1, 1, 151936, 2),
    (3, 4, 151936, 8), (40, 8, 10007, 16),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(SIZES)))
def test_matches_64_bits(case, dtype):
    G, K, V, count = SIZES[case]
    check(*make(G, K, V, dtype, seed=case), count)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pitch,offset", [(1, 0), (3, 1), (0, 5), (7, 7), (8, 0)])
def test_rows_at_any_address(pitch, offset, dtype):
    """What lies between the rows is NaN."""
    check(*make(2, 3, 5003, dtype, seed=pitch, pitch=pitch, offset=offset), 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9, 2048, 30000])
def test_equal_sums_go_to_the_lowest_beam_and_token(V, dtype):
    logits = torch.zeros((8, V), dtype=dtype, device="cuda")
    logits[:, V // 2] = -0.0
    scores = torch.tensor([[-1.0] * 4, [-1.0, -2.0, -1.0, -1.0]], device="cuda")
    _, parents, tokens = check(logits, scores, 8)
    assert tokens.tolist() == [list(range(8))] * 2 and not bool(parents.any())
    one = torch.full((3, V), -5.0, dtype=dtype, device="cuda")
    one[:, [V - 1, 3, 5]] = 2.0
    _, parents, tokens = check(one, torch.zeros((1, 3), device="cuda"), 7)
    assert tokens[0].tolist() == [3, 5, V - 1] * 2 + [3] and parents[0].tolist() == [0, 0, 0, 1, 1, 1, 2]


@pytest.mark.parametrize("order", ["rising", "falling", "blocks", "one thread", "one warp"])
@pytest.mark.parametrize("count", [1, 16, 64])
def test_values_in_unlucky_orders(order, count):
    """Every logit beats the ones before it; all large ones fall to few threads or warps."""
    V = 60000
    i = torch.arange(V, dtype=torch.float64)
    x = {"rising": i / V, "falling": 1 - i / V, "blocks": (i // 8192) + (i % 64) / 64,
         "one thread": torch.where((i // 4) % 256 == 7, i / V + 1, -i / V),
         "one warp": torch.where((i // 128) % 8 == 3, i / V, i / V - 9)}[order]
    x = torch.stack([x, x.flip(0)]).float().cuda()
    check(x, torch.tensor([[-3.0, -3.5]], device="cuda"), count)


def test_beams_and_tokens_that_are_out():
    logits, scores = make(3, 4, 6000, seed=21)
    logits[:, 100:5000] = -INF  # banned
    scores[0, 1:] = -INF  # the first step: of beams that are alike one counts
    scores[1] = -INF  # nothing left
    scores[2, 0] = float("nan")
    scores[2, 1] = INF
    logits[10, 50] = float("nan")
    logits[11, 5999] = INF
    _, parents, _ = check(logits, scores, 8)
    assert not bool(parents[0].any()) and parents[1].tolist() == parents[2].tolist() == [-1] * 8
    logits, scores = make(1, 3, 3000, seed=22)
    logits[0] = -INF  # no token
    logits[1] = float("nan")
    logits[2, 3:] = -INF  # three of them
    _, parents, tokens = check(logits, scores, 6)
    assert parents[0].tolist() == [2, 2, 2, -1, -1, -1] and sorted(tokens[0, :3].tolist()) == [0, 1, 2]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_of_the_lowest_value_and_large_logits(dtype):
    logits, scores = make(2, 2, 4000, dtype, seed=23)
    logits[:, 5:] = torch.finfo(dtype).min
    check(logits, scores, 4)
    logits, scores = make(2, 2, 4000, dtype, seed=24)
    logits *= 1000  # all but one probability vanish
    check(logits, scores, 8, exactly=dtype is torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_nothing_but_masks_and_logits_of_any_size(dtype):
    """Whole rows at the type's lowest value (all tokens alike), rows far from zero, such parts among others."""
    V = 40000
    low = torch.finfo(dtype).min
    logits, scores = make(1, 8, V, dtype, seed=31)
    logits[0] = low
    logits[1] = -low
    logits[2, 1000:] = low
    logits[3, :20000], logits[3, 20000:] = low, low / 2
    logits[4] = logits[4] * 8 + 2.0 ** 22  # fp32: steps of a half; bf16: all alike
    logits[5] = logits[5] - 2.0 ** 21
    logits[6] = logits[6] * 1e6  # bf16: steps of thousands
    logits[7, :100] = 1e30
    for beams in range(8):  # one by one, and all together
        check(logits[beams:beams + 1], scores[:, beams:beams + 1], 16)
    scores = torch.zeros((1, 8), device="cuda") - torch.arange(8, device="cuda") / 3
    check(logits, scores, 64)


def test_sums_that_64_bits_do_not_tell_apart():
    """Scores so large that the logits are lost in the sums: the lowest beam first, its tokens as their logits."""
    x, _ = make(2, 3, 5000, seed=40)
    scores = torch.tensor([[-1e30, -1e30, -1e30], [-1e30, -1e29, -2e30]], device="cuda")
    order = x.cpu().argsort(dim=1, descending=True, stable=True)
    values, parents, tokens = (t.cpu() for t in ops.beam_select(x, scores, 40))
    assert parents.tolist() == [[0] * 40, [1] * 40]
    assert torch.equal(tokens[0], order[0, :40]) and torch.equal(tokens[1], order[4, :40])
    assert torch.equal(values, torch.tensor([[-1e30] * 40, [-1e29] * 40]))


def test_scores_between_rows_of_a_wider_tensor():
    logits, scores = make(4, 3, 2500, seed=25)
    wide = torch.full((4, 9), 7.0, device="cuda")
    wide[:, 2:5] = scores
    check(logits, wide[:, 2:5], 6)


def test_many_groups():
    check(*make(1500, 2, 300, seed=26), 4, exactly=False)


def test_repeatable_graph_and_streams():
    logits, scores = make(6, 5, 50257, seed=27)
    want = ops.beam_select(logits, scores, 10)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, ops.beam_select(logits, scores, 10)))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out1 = ops.beam_select(logits, scores, 10)
    with torch.cuda.graph(g2):
        out2 = ops.beam_select(logits, scores, 10)
    for seed in (28, 29, 27):
        x, s = make(6, 5, 50257, seed=seed)
        logits.copy_(x)
        scores.copy_(s)
        torch.cuda.synchronize()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        for _ in range(5):
            with torch.cuda.stream(s1):
                g1.replay()
            with torch.cuda.stream(s2):
                g2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out1, out2))
        best, p, t, _ = exact(logits, scores, 10)
        assert torch.equal(out1[1].cpu(), p) and torch.equal(out1[2].cpu(), t)
    assert all(torch.equal(a, b) for a, b in zip(want, out1))


def test_refuses():
    logits, scores = make(2, 3, 100)
    with pytest.raises(TypeError):
        ops.beam_select(logits.half(), scores, 4)
    with pytest.raises(TypeError):
        ops.beam_select(logits, scores.double(), 4)
    with pytest.raises(ValueError, match="groups"):
        ops.beam_select(logits[:5], scores, 4)
    with pytest.raises(ValueError, match="contiguous"):
        ops.beam_select(logits.t().contiguous().t(), scores, 4)
    for count, n in ((0, 100), (65, 100), (-1, 100), (4, 0)):
        with pytest.raises(ops._lib.XbError):
            ops.beam_select(logits[:, :n], scores, count)
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_select(logits.cpu(), scores, 4)
    values, parents, tokens = ops.beam_select(logits[:0], scores[:0], 4)
    assert values.shape == parents.shape == tokens.shape == (0, 4)
