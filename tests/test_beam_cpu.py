"""Beam search without a GPU: argument checks of the selection's C entry points, and the search over a paged cache."""

import ctypes
import math

import pytest
import torch

from xb200 import _lib, ops
from xb200._lib import XbError
from xb200.beam import generate_beams
from xb200.paged import PagedKVCache


def _select(**kw):
    a = dict(logits=1 << 12, scores=1 << 13, groups=2, beams=4, vocab=1000, ld=1000, ld_scores=4, count=8, dtype=1,
             values=1 << 14, parents=1 << 15, tokens=1 << 16, ws=None, ws_bytes=0)
    a.update(kw)
    _lib.call("xb_beam_select", *a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(groups=-1), _lib.XB_ERR_INVALID, "shape"),
    (dict(beams=0), _lib.XB_ERR_INVALID, "shape"),
    (dict(vocab=0), _lib.XB_ERR_INVALID, "shape"),
    (dict(count=0), _lib.XB_ERR_INVALID, "shape"),
    (dict(count=-3), _lib.XB_ERR_INVALID, "shape"),
    (dict(beams=65), _lib.XB_ERR_UNSUPPORTED, "64 beams"),
    (dict(count=65), _lib.XB_ERR_UNSUPPORTED, "64 continuations"),
    (dict(groups=(1 << 20) + 1), _lib.XB_ERR_UNSUPPORTED, "groups"),
    (dict(vocab=1 << 31, ld=1 << 31), _lib.XB_ERR_UNSUPPORTED, "tokens"),
    (dict(dtype=2), _lib.XB_ERR_UNSUPPORTED, "dtype"),
    (dict(logits=None), _lib.XB_ERR_INVALID, "null"),
    (dict(scores=None), _lib.XB_ERR_INVALID, "null"),
    (dict(tokens=None), _lib.XB_ERR_INVALID, "null"),
    (dict(ld=999), _lib.XB_ERR_INVALID, "pitch"),
    (dict(ld_scores=3), _lib.XB_ERR_INVALID, "pitch"),
    (dict(logits=4098), _lib.XB_ERR_UNSUPPORTED, "aligned"),
    (dict(), _lib.XB_ERR_INVALID, "workspace"),
    (dict(ws=1 << 20, ws_bytes=64), _lib.XB_ERR_INVALID, "workspace"),
    (dict(ws=(1 << 20) + 8, ws_bytes=1 << 30), _lib.XB_ERR_INVALID, "workspace"),
])
def test_beam_select_refuses(kw, code, text):
    with pytest.raises(XbError) as e:
        _select(**kw)
    assert e.value.code == code and text in e.value.message, e.value.message


def test_beam_select_without_groups_is_a_no_op():
    _select(groups=0, logits=None, scores=None, values=None)


def test_workspace_size():
    need = ctypes.c_size_t(0)
    _lib.call("xb_beam_select_workspace_size", 0, 4, 1000, 8, ctypes.byref(need))
    assert need.value == 0
    for groups in (1, 4, 40, 4000):
        _lib.call("xb_beam_select_workspace_size", groups, 4, 151936, 8, ctypes.byref(need))
        parts = need.value // (groups * 4 * (8 * 8 + 16))  # a list and the sums of each part of a row
        assert need.value == groups * 4 * parts * (8 * 8 + 16) and 1 <= parts <= 38


# ----------------------------------------------------------------------------- the search, on a model of tables


class _Cfg:
    n_layer, n_kv_head, head_dim = 1, 1, 16


class _Table:
    """A model whose logits depend on the tokens so far, which it finds in the cache's pages: what the cache shares,
    forks and frees has to be right for the search to be."""

    position_limit, device, cfg = 64, torch.device("cpu"), _Cfg

    def __init__(self, vocab, seed, end_bias=0.0):
        self.vocab, self.seed, self.end_bias = vocab, seed, end_bias
        self.steps = 0

    def logits(self, tokens):
        g = torch.Generator().manual_seed(hash((self.seed, *tokens)) & 0x7FFFFFFF)
        x = torch.randn(self.vocab, generator=g) * 2
        x[0] += self.end_bias
        return x

    def forward_paged(self, ids, cache, seqs, counts=None, next_token=None):
        self.steps += 1
        batch = cache.step(seqs, counts)
        start, P = batch.q_start.tolist(), cache.page_size
        out = []
        for i, q in enumerate(seqs):
            for t in range(start[i], start[i + 1]):
                p = int(batch.positions[t])
                cache.pages[0, 0, int(batch.page_table[i, p // P]), 0, p % P, 0] = int(ids[t])
            out.append(self.logits([int(cache.pages[0, 0, cache.page_ids(q)[p // P], 0, p % P, 0])
                                    for p in range(cache.length(q))]))
        return torch.stack(out)


def _plain_select(logits, scores, count):
    G, K = scores.shape
    total = scores.view(-1, 1) + torch.log_softmax(logits, 1)
    total = torch.where(total.isfinite(), total, -math.inf).view(G, -1)
    best, at = total.sort(dim=1, descending=True, stable=True)
    V = logits.shape[1]
    pad = max(0, count - best.shape[1])
    best = torch.nn.functional.pad(best[:, :count], (0, pad), value=-math.inf)
    at = torch.nn.functional.pad(at[:, :count], (0, pad))
    none = best == -math.inf
    return best, (at // V).masked_fill(none, -1), (at % V).masked_fill(none, -1)


@pytest.fixture
def plain(monkeypatch):
    def copy(pages, src, dst, dim=2):
        pages[:, :, dst] = pages[:, :, src]

    monkeypatch.setattr(ops, "copy_pages", copy)
    monkeypatch.setattr(ops, "beam_select", _plain_select)


def _search(model, prompt, K, steps, end, penalty):
    """The same search on lists."""
    live, done = [([], 0.0)], []
    for _ in range(steps):
        c = []
        for b, (toks, s) in enumerate(live):
            lp = torch.log_softmax(model.logits(prompt + toks), 0)
            c += [(torch.tensor(s, dtype=torch.float32) + lp[v], -(b * model.vocab + v), toks + [v])
                  for v in range(model.vocab)]
        c.sort(key=lambda x: (-float(x[0]), -x[1]))
        live, more = [], c[:2 * K]
        for rank, (s, _, toks) in enumerate(more):
            if len(live) == K:
                break
            if toks[-1] == end:
                if rank < K:
                    done.append((float(s) / len(toks) ** penalty, toks))
            else:
                live.append((toks, float(s)))
        done.sort(key=lambda x: -x[0])
        done = done[:K]
        if not live or (len(done) == K and done[-1][0] >= live[0][1] / len(live[0][0]) ** penalty):
            live = []
            break
    done += [(s / len(t) ** penalty, t) for t, s in live]
    return sorted(done, key=lambda x: -x[0])[:K]


@pytest.mark.parametrize("page", [8, 16])
@pytest.mark.parametrize("K,steps,end,penalty,bias", [(1, 7, None, 1.0, 0), (3, 9, None, 1.0, 0), (4, 12, 0, 1.0, 0),
                                                      (4, 12, 0, 0.0, 3), (2, 20, 0, 2.0, 1), (5, 1, 0, 1.0, 2),
                                                      (32, 4, 0, 1.0, 0)])
def test_search_matches_a_search_on_lists(plain, K, steps, end, penalty, bias, page):
    model = _Table(11, seed=K, end_bias=bias)
    prompts = [[3, 1, 4, 1, 5], [2], list(range(1, 11)) * 2, [7] * 8]
    need = sum(len(p) // page + K * -(-(len(p) % page + steps - 1) // page) for p in prompts)
    cache = PagedKVCache(_Cfg, need, page, device="cpu")
    got = generate_beams(model, [torch.tensor(p) for p in prompts], K, steps, end, penalty, cache=cache, graph=False)
    assert cache.free_pages == need and len(cache) == 0
    for p, h in zip(prompts, got):
        want = _search(model, p, K, steps, end, penalty)
        assert [x.tokens for x in h] == [t for _, t in want]
        for x, (score, t) in zip(h, want):
            assert abs(x.score - score) < 1e-4 and abs(x.logprob - score * len(t) ** penalty) < 1e-3


def test_one_beam_is_greedy(plain):
    model = _Table(50, seed=9)
    (h,), = generate_beams(model, [torch.tensor([5, 6])], 1, 6, graph=False)
    tokens = []
    for _ in range(6):
        tokens.append(int(model.logits([5, 6] + tokens).argmax()))
    assert h.tokens == tokens


def test_fewer_continuations_than_beams(plain):
    """Two tokens and five beams: places are left over in the first steps."""
    model = _Table(2, seed=4)
    got, = generate_beams(model, [torch.tensor([1])], 5, 4, graph=False)
    want = _search(model, [1], 5, 4, None, 1.0)
    assert [h.tokens for h in got] == [t for _, t in want]
    only_end = _Table(1, seed=4)
    got, = generate_beams(only_end, [torch.tensor([0])], 3, 4, end_token=0, graph=False)
    assert [h.tokens for h in got] == [[0]] and only_end.steps == 1


def test_search_refuses(plain):
    model = _Table(5, seed=1)
    one = torch.tensor([1])
    for args in (([one], 0, 3), ([one], 33, 3), ([], 2, 3), ([one], 2, 0), ([torch.tensor([[1]])], 2, 3),
                 ([torch.ones(60, dtype=torch.int64)], 2, 6)):
        with pytest.raises(ValueError):
            generate_beams(model, *args, graph=False)
    with pytest.raises(ValueError, match="multiple of 8"):
        generate_beams(model, [one], 2, 3, page_size=12, graph=False)
    cache = PagedKVCache(_Cfg, 3, 8, device="cpu")
    with pytest.raises(RuntimeError, match="full"):
        generate_beams(model, [one], 4, 9, cache=cache, graph=False)
    assert cache.free_pages == 3 and len(cache) == 0


def test_reorder_keeps_the_books(plain):
    c = PagedKVCache(_Cfg, 20, 8, device="cpu")
    a, b, d = c.add(), c.add(), c.add()
    c.step([a, b, d], [9, 9, 9])
    new = c.reorder([a, b, d], [2, 2, 0, 2])
    assert new[0] == d and new[2] == a and len(set(new)) == 4 and len(c) == 4
    assert c.page_ids(new[1]) == c.page_ids(d) == c.page_ids(new[3]) and c.free_pages == 16
    with pytest.raises(KeyError):
        c.length(b)
    for seqs, parents in (([a, a], [0, 1]), ([a, d], [2]), ([a, d], [-1])):
        with pytest.raises(ValueError):
            c.reorder(seqs, parents)
    with pytest.raises(KeyError):
        c.reorder([a, 99], [0])
    assert len(c) == 4 and c.reorder(new, []) == [] and c.free_pages == 20 and len(c) == 0
