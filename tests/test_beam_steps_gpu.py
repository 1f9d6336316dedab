"""A beam search put together from its parts (a graph that gives logits, the choice, the
cache's books), as the documentation shows it."""

import pytest
import torch
from test_paged_models_gpu import _ids, gpt2, qwen  # noqa: F401 (fixtures)

from xb200 import ops
from xb200.paged import PagedDecodeGraph, PagedKVCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
@pytest.mark.parametrize("family", ["qwen", "gpt2"])
def test_a_search_of_ones_own(family, dtype, request):
    m = request.getfixturevalue(family)
    model = m[0] if family == "qwen" else m
    prompts = [_ids(n, model.cfg.vocab_size, 140 + n) for n in (30, 9)]
    K, steps, G = 4, 6, len(prompts)
    cache = PagedKVCache(model.cfg, 64, 16, dtype=dtype)
    told = [[[] for _ in range(1)] for _ in prompts]

    seqs = [cache.add() for _ in prompts]
    logits = model.forward_paged(torch.cat(prompts).cuda(), cache, seqs, [len(p) for p in prompts])
    beams, scores = [[q] for q in seqs], torch.zeros((G, 1), device="cuda")
    graph = PagedDecodeGraph(model, cache, batch=G * K, max_positions=64, logits=True)
    for step in range(steps):
        scores, parents, tokens = ops.beam_select(logits, scores, K)
        beams = [cache.reorder(s, p) for s, p in zip(beams, parents.tolist())]
        told = [[t[p] + [x] for p, x in zip(ps, xs)] for t, ps, xs in zip(told, parents.tolist(), tokens.tolist())]
        if step + 1 < steps:
            logits = graph.step([q for s in beams for q in s], tokens.flatten())

    want = model.generate_beams(prompts, K, steps, dtype=dtype)
    assert told == [[h.tokens for h in hyps] for hyps in want]
    assert scores.tolist() == [[h.logprob for h in hyps] for hyps in want]
    for q in sum(beams, []):
        cache.free(q)
    assert cache.free_pages == 64 and ops.device_status() == 0 and ops.page_status() == 0
