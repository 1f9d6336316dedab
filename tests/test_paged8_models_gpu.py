"""Qwen2.5 and GPT-2 over 8-bit paged caches, and beam search over all of them.

Layer 0 sees the same inputs whatever the cache holds, so its codes are those of
the bf16 cache's numbers, bit for bit.  Logits: a code is off by at most 2^-4 of its
number (e4m3; int8 2^-7 of the vector's largest), so an attention output by about as
much, and after two layers the residual stream by at most 2 x 2^-4 of its
length: the cosine stays above 1 - (2^-3)^2 / 2 = 0.992.
"""

import pytest
import torch
from test_paged8_gpu import quantise, values
from test_paged_models_gpu import _ids, gpt2, qwen  # noqa: F401 (fixtures)

from xb200 import ops
from xb200.paged import PagedDecodeGraph, PagedKVCache

pytestmark = pytest.mark.gpu

DTYPES = [torch.int8, torch.float8_e4m3fn]


def _model(request, family):
    m = request.getfixturevalue(family)
    return m[0] if family == "qwen" else m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("family", ["qwen", "gpt2"])
def test_steps_over_8_bit_pages(family, dtype, request):
    """Prompts, a step of a chunk and single tokens, single tokens; forks, a compaction, reading back."""
    model = _model(request, family)
    V = model.cfg.vocab_size
    caches = [PagedKVCache(model.cfg, 60, 16, dtype=d) for d in (torch.bfloat16, dtype)]
    held = [[c.add() for _ in range(3)] for c in caches]
    for step, counts in enumerate(([200, 37, 5], [90, 1, 1], [1, 1, 1])):
        ids = _ids(sum(counts), V, 40 + step).cuda()
        a, b = (model.forward_paged(ids, c, h, counts).double() for c, h in zip(caches, held))
        assert torch.nn.functional.cosine_similarity(a, b, dim=-1).min().item() >= 0.992
    want_k, want_v = caches[0].read(held[0], 0)
    got_k, got_v = caches[1].read(held[1], 0)
    assert got_k.shape == (291 + 39 + 7, model.cfg.n_kv_head, 64)
    for got, want in ((got_k, want_k), (got_v, want_v)):
        assert torch.equal(got.cpu().double(), values(*quantise(want.cpu(), dtype)))
    c, (s0, s1, s2) = caches[1], held[1]
    fork = c.fork(s1)
    c.free(s0)
    toks = torch.tensor([3, 4, 5], device="cuda")
    before = model.forward_paged(toks, c, [s1, s2, fork])
    for s in (s1, s2, fork):
        c.truncate(s, c.length(s) - 1)
    assert c.compact() > 0
    assert torch.equal(model.forward_paged(toks, c, [s1, s2, fork]), before)
    k, v = c.read([fork], model.cfg.n_layer - 1)
    k1, v1 = c.read([s1], model.cfg.n_layer - 1)
    assert k.shape[0] == 40 and torch.equal(k[:39], k1[:39]) and torch.equal(v[:39], v1[:39])
    assert c.read([], 0)[0].shape == (0, model.cfg.n_kv_head, 64)
    assert ops.device_status() == 0 and ops.page_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_graph_serves_every_step(dtype, request):
    model = _model(request, "qwen")
    V = model.cfg.vocab_size
    cache, eager = (PagedKVCache(model.cfg, 60, 16, dtype=dtype) for _ in range(2))
    prompts = [_ids(n, V, 70 + n) for n in (5, 40, 130)]
    graphs = [PagedDecodeGraph(model, cache, 2, 200), PagedDecodeGraph(model, cache, 2, 200, logits=True)]
    handles = []
    for c in (cache, eager):
        seqs = [c.add() for _ in prompts]
        model.forward_paged(torch.cat(prompts).cuda(), c, seqs, [p.numel() for p in prompts])
        handles.append(seqs)
    toks = torch.tensor([11, 12], device="cuda")
    for i, pair in enumerate(([0, 1], [2, 1], [1, 0], [2, 0], [2, 1])):
        got = graphs[i % 2].step([handles[0][j] for j in pair], toks)
        want = model.forward_paged(toks, eager, [handles[1][j] for j in pair])
        assert torch.equal(got, want.argmax(-1) if i % 2 == 0 else want)
        toks = want.argmax(-1)
    assert ops.device_status() == 0 and ops.page_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("family", ["qwen", "gpt2"])
def test_generation(family, dtype, request):
    model = _model(request, family)
    prompts = [_ids(n, model.cfg.vocab_size, 90 + n) for n in (24, 7, 1)]
    out = model.generate_paged(prompts, 6, dtype=dtype)
    assert torch.equal(out, model.generate_paged(prompts, 6, graph=False, dtype=dtype))
    cache = PagedKVCache(model.cfg, 12, 16, dtype=dtype)
    assert torch.equal(out, model.generate_paged(prompts, 6, cache=cache)) and cache.free_pages == 12


def _rescored(model, prompt, tokens, dtype):
    """log-probabilities of a continuation, by one packed step of a cache of its own."""
    cache = PagedKVCache(model.cfg, 64, 16, dtype=dtype)
    total, seq = 0.0, cache.add()
    logits = model.forward_paged(prompt.cuda(), cache, [seq], [prompt.numel()])
    for t in tokens:
        total += float(torch.log_softmax(logits.double(), -1)[0, t])
        logits = model.forward_paged(torch.tensor([t], device="cuda"), cache, [seq])
    return total


@pytest.mark.parametrize("dtype", [torch.bfloat16, *DTYPES])
@pytest.mark.parametrize("family", ["qwen", "gpt2"])
def test_beams(family, dtype, request):
    """Continuations with the sums that they claim, as good as the greedy one's at least; the same with and without a graph.

    The steps of a search and of the rescoring split their sums differently: logits agree to 2 % of their range
    (test_paged_models_gpu.py), far more closely in the mean."""
    model = _model(request, family)
    prompts = [_ids(n, model.cfg.vocab_size, 95 + n) for n in (33, 7, 1)]
    steps, K = 6, 4
    got = model.generate_beams(prompts, K, steps, dtype=dtype)
    assert got == model.generate_beams(prompts, K, steps, dtype=dtype, graph=False)
    greedy = model.generate_paged(prompts, steps, dtype=dtype).tolist()
    for p, hyps, g in zip(prompts, got, greedy):
        assert len(hyps) == K and len({tuple(h.tokens) for h in hyps}) == K
        assert all(len(h.tokens) == steps and abs(h.score * steps - h.logprob) < 1e-9 for h in hyps)
        assert [h.score for h in hyps] == sorted((h.score for h in hyps), reverse=True)
        slack = 0.02 * steps
        assert abs(_rescored(model, p, hyps[0].tokens, dtype) - hyps[0].logprob) <= slack
        assert hyps[0].logprob >= _rescored(model, p, g, dtype) - slack
    assert ops.device_status() == 0 and ops.page_status() == 0


def test_one_beam_is_the_greedy_continuation(request):
    """Up to near ties: the tokens are the argmax of the same kernels' logits."""
    model = _model(request, "qwen")
    prompts = [_ids(n, model.cfg.vocab_size, 120 + n) for n in (20, 3)]
    got = model.generate_beams(prompts, 1, 5)
    assert [h[0].tokens for h in got] == model.generate_paged(prompts, 5).tolist()


def test_beams_that_end(request):
    """The token that all searches choose second ends them: finished ones and longer ones are ranked together."""
    model = _model(request, "gpt2")
    prompt = _ids(12, model.cfg.vocab_size, 130)
    first = model.generate_beams([prompt], 3, 8)[0]
    end = first[0].tokens[2]
    cache = PagedKVCache(model.cfg, 40, 8)
    got = model.generate_beams([prompt, prompt[:5]], 3, 8, end_token=end, length_penalty=0.5, cache=cache)
    assert cache.free_pages == 40 and len(cache) == 0
    for hyps in got:
        assert 1 <= len(hyps) <= 3
        for h in hyps:
            assert end not in h.tokens[:-1] and (len(h.tokens) == 8 or h.tokens[-1] == end)
            assert abs(h.score - h.logprob / len(h.tokens) ** 0.5) < 1e-9
    assert any(h.tokens[-1] == end for h in got[0])
