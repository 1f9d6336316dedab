"""Qwen2.5 and GPT-2 over a paged cache: the models' own contiguous path and
the oracles as references, with the tolerances of the contiguous model tests
(tests/test_qwen_gpu.py: logits reach cosine 0.9999 and stay within 2 % of
their range at two layers)."""

import pytest
import torch

from oracle.qwen import OracleQwen
from xb200 import ops
from xb200.gpt2 import GPT2Config, GPT2Model
from xb200.gpt2 import random_weights as gpt2_weights
from xb200.paged import PagedDecodeGraph, PagedKVCache
from xb200.qwen import Qwen2Model, QwenConfig, random_weights

pytestmark = pytest.mark.gpu


def _close(got, ref, cos_min=0.9999, rel=0.02):
    got, ref = got.double().cpu(), ref.double().cpu()
    cos = torch.nn.functional.cosine_similarity(got, ref, dim=-1).min().item()
    assert cos >= cos_min and (got - ref).abs().max().item() <= rel * ref.abs().max().item(), cos


def _ids(n, vocab, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed))


@pytest.fixture(scope="module")
def qwen():
    cfg = QwenConfig(n_layer=2)
    sd = random_weights(cfg, seed=31)
    return Qwen2Model(sd, cfg, rope_len=1024), OracleQwen(sd, cfg)


@pytest.fixture(scope="module")
def gpt2():
    cfg = GPT2Config(n_layer=2)
    return GPT2Model(gpt2_weights(cfg, seed=32), cfg)


def _contiguous(model, ids):
    """Logits after the last of `ids`, by the model's contiguous path."""
    return model.forward(ids.view(1, -1).cuda(), model.new_cache(1, ids.numel()), last_only=True)


def test_prompts_chunks_and_single_tokens_match_the_oracle(qwen):
    """Three sequences: packed prompts, then a step that mixes a chunk and single tokens, then single tokens."""
    model, orc = qwen
    V = model.cfg.vocab_size
    total = [40, 9, 23]
    ids = [_ids(n, V, 40 + i) for i, n in enumerate(total)]
    cache = PagedKVCache(model.cfg, 16, 8)
    seqs = [cache.add() for _ in total]
    at = [0, 0, 0]
    for counts in ([20, 7, 21], [19, 1, 1], [1, 1, 1]):
        packed = torch.cat([ids[i][at[i]:at[i] + n] for i, n in enumerate(counts)])
        got = model.forward_paged(packed.cuda(), cache, seqs, counts)
        at = [a + n for a, n in zip(at, counts)]
        for i in range(3):
            ref = orc.forward(ids[i][None, :at[i]], orc.new_cache(1, at[i]))[0, -1]
            _close(got[i:i + 1], ref[None])
    assert [cache.length(s) for s in seqs] == total
    assert ops.device_status() == 0 and ops.page_status() == 0 and ops.token_status() == 0


@pytest.mark.parametrize("family", ["qwen", "gpt2"])
def test_large_steps_match_the_contiguous_path(family, request):
    model = request.getfixturevalue("qwen")[0] if family == "qwen" else request.getfixturevalue("gpt2")
    V = model.cfg.vocab_size
    a, b = _ids(300, V, 50), _ids(77, V, 51)
    cache = PagedKVCache(model.cfg, 40, 16)
    sa, sb = cache.add(), cache.add()
    _close(model.forward_paged(torch.cat([a[:200], b[:60]]).cuda(), cache, [sa, sb], [200, 60])[1:],
           _contiguous(model, b[:60]))
    got = model.forward_paged(torch.cat([b[60:], a[200:]]).cuda(), cache, [sb, sa], [17, 100])
    _close(got, torch.cat([_contiguous(model, b), _contiguous(model, a)]))
    nxt = torch.empty(2, dtype=torch.int64, device="cuda")
    one = torch.tensor([5, 9], device="cuda")
    assert model.forward_paged(one, cache, [sa, sb], next_token=nxt) is None
    cache.truncate(sa, 300)
    cache.truncate(sb, 77)
    logits = model.forward_paged(one, cache, [sa, sb])
    assert torch.equal(nxt, logits.argmax(-1))
    assert ops.device_status() == 0 and ops.page_status() == 0


def test_forked_sequences_diverge_and_keep_their_past(qwen):
    model, _ = qwen
    V = model.cfg.vocab_size
    prompt = _ids(21, V, 60)  # ends inside a page
    tails = [_ids(5, V, 61 + i) for i in range(3)]
    cache = PagedKVCache(model.cfg, 20, 16)
    root = cache.add()
    model.forward_paged(prompt.cuda(), cache, [root], [21])
    seqs = [root, cache.fork(root), cache.fork(root)]
    for i in range(5):
        got = model.forward_paged(torch.stack([t[i] for t in tails]).cuda(), cache, seqs)
    for k in range(3):
        _close(got[k:k + 1], _contiguous(model, torch.cat([prompt, tails[k]])))
    # a compaction moves pages, not results
    cache.free(seqs[0])
    before = model.forward_paged(torch.tensor([3, 4]).cuda(), cache, seqs[1:])
    for s in seqs[1:]:
        cache.truncate(s, 26)
    assert cache.compact() > 0
    assert torch.equal(model.forward_paged(torch.tensor([3, 4]).cuda(), cache, seqs[1:]), before)


def test_one_graph_serves_every_step(qwen):
    """Replays for sequences of different lengths that change between steps equal eager steps, bit for bit."""
    model, _ = qwen
    V = model.cfg.vocab_size
    cache, eager = (PagedKVCache(model.cfg, 60, 16) for _ in range(2))
    prompts = [_ids(n, V, 70 + n) for n in (5, 40, 130)]
    graph = PagedDecodeGraph(model, cache, 2, 200)
    handles = []
    for c in (cache, eager):
        seqs = [c.add() for _ in prompts]
        model.forward_paged(torch.cat(prompts).cuda(), c, seqs, [p.numel() for p in prompts])
        handles.append(seqs)
    toks = torch.tensor([11, 12], device="cuda")
    for pair in ([0, 1], [2, 1], [1, 0], [2, 0], [2, 1]):
        got = graph.step([handles[0][i] for i in pair], toks)
        want = torch.empty_like(got)
        model.forward_paged(toks, eager, [handles[1][i] for i in pair], next_token=want)
        assert torch.equal(got, want)
        # larger work in between: the graph's scratch is its own
        big = eager.add()
        model.forward_paged(_ids(90, V, 80).cuda(), eager, [big], [90], next_token=torch.empty(1, dtype=torch.int64,
                                                                                               device="cuda"))
        eager.free(big)
        toks = want.clone()
    for a, b in zip(*handles):
        assert cache.length(a) == eager.length(b)
    with pytest.raises(ValueError, match="captured for 2"):
        graph.step(handles[0][:1], toks[:1])
    assert ops.device_status() == 0 and ops.page_status() == 0


@pytest.mark.parametrize("family", ["qwen", "gpt2"])
def test_generate_paged_equals_generate_for_equal_lengths(family, request):
    """Tokens of the contiguous generation, up to the first near-tie of a sequence."""
    model = request.getfixturevalue("qwen")[0] if family == "qwen" else request.getfixturevalue("gpt2")
    ids = torch.stack([_ids(24, model.cfg.vocab_size, 90 + i) for i in range(3)])
    want, _ = model.generate(ids.cuda(), 6)
    got = model.generate_paged(list(ids), 6)
    assert got.shape == (3, 6) and torch.equal(got[:, 0], want[:, 0])
    assert torch.equal(got, model.generate_paged(list(ids), 6, graph=False))
    mixed = [ids[0], ids[1][:7], ids[2][:1]]
    cache = PagedKVCache(model.cfg, 12, 16)
    out = model.generate_paged(mixed, 4, cache=cache)
    assert out.shape == (3, 4) and cache.free_pages == 12 and len(cache) == 0
    for i, p in enumerate(mixed):
        logits = _contiguous(model, p)[0]
        top = logits.max()
        assert float(top - logits[out[i, 0]]) <= 0.04 * float(logits.abs().max())


def test_forward_paged_refusals(qwen, gpt2):
    model, _ = qwen
    cache = PagedKVCache(model.cfg, 4, 16)
    a = cache.add()
    with pytest.raises(ValueError, match="1-D"):
        model.forward_paged(torch.zeros((1, 2), dtype=torch.int64, device="cuda"), cache, [a], [2])
    with pytest.raises(ValueError, match="tokens"):
        model.forward_paged(torch.zeros(3, dtype=torch.int64, device="cuda"), cache, [a], [2])
    with pytest.raises(RuntimeError, match="full"):
        model.forward_paged(torch.zeros(65, dtype=torch.int64, device="cuda"), cache, [a], [65])
    with pytest.raises(ValueError, match="RoPE table"):
        model.forward_paged(torch.zeros(1025, dtype=torch.int64, device="cuda"), cache, [a], [1025])
    assert cache.length(a) == 0 and cache.free_pages == 4
    other = PagedKVCache(gpt2.cfg, 4, 16)
    with pytest.raises(ValueError, match="position table"):
        gpt2.forward_paged(torch.zeros(1025, dtype=torch.int64, device="cuda"), other, [other.add()], [1025])
    with pytest.raises(ValueError, match="max_positions"):
        PagedDecodeGraph(model, cache, 1, 1025)
    with pytest.raises(ValueError):
        model.generate_paged([], 3)
    with pytest.raises(ValueError):
        model.generate_paged([torch.zeros(0, dtype=torch.int64)], 3)



def test_refused_steps_leave_the_cache_as_it_was(qwen, gpt2):
    """What the operators of a step would refuse is refused before the cache gives room for it."""
    model, _ = qwen
    cache = PagedKVCache(model.cfg, 4, 16)
    a = cache.add()
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    one = torch.zeros(1, dtype=torch.int64, device="cuda")
    for kw in (dict(ids=ids.int()), dict(ids=ids.cpu()), dict(next_token=one.int()), dict(next_token=one.cpu()),
               dict(next_token=ids), dict(next_token=torch.zeros((1, 1), dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            model.forward_paged(**{"ids": ids, "cache": cache, "seqs": [a], "counts": [3], **kw})
    other = PagedKVCache(gpt2.cfg, 4, 16)
    b = other.add()
    with pytest.raises(ValueError, match="another model"):
        model.forward_paged(ids, other, [b], [3])
    with pytest.raises(ValueError, match="another model"):
        PagedDecodeGraph(model, other, 1, 64)
    graph = PagedDecodeGraph(model, cache, 1, 64)
    with pytest.raises(ValueError, match="int64"):
        graph.step([a], one.float())
    assert cache.length(a) == other.length(b) == 0 and cache.free_pages == other.free_pages == 4


def test_generation_up_to_the_last_position(qwen):
    """A prompt and its continuation may fill the table: the last token is never fed back."""
    model, _ = qwen
    prompt = _ids(1024 - 4, model.cfg.vocab_size, 95)
    cache = PagedKVCache(model.cfg, 64, 16)  # 1024 positions
    out = model.generate_paged(iter([prompt]), 5, cache=cache)
    assert torch.equal(out, model.generate_paged([prompt], 5, graph=False)) and cache.free_pages == 64
    with pytest.raises(ValueError, match="positions"):
        model.generate_paged([prompt], 6)
