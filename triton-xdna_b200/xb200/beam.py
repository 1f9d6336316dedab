"""Beam search over a paged KV cache.

The reference generates greedily (examples/qwen2_5/model.py:1134-1179,
examples/gpt2/model.py:1144-1206); here each prompt keeps `beams` unfinished
continuations, the likeliest ones.  A beam is a sequence of the cache: beams of one prompt
share the pages of what they have in common, going on from another beam is a
fork, and only the page that two of them write into is copied.  A step is one
replay of a decode graph for all beams of all prompts and one
``ops.beam_select`` over their logits; which beam goes on from which is settled
on the host, where the cache's books are.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops
from .paged import PagedDecodeGraph, PagedKVCache, check_prompts


@dataclass
class Hypothesis:
    """A continuation: its tokens (the end token included, if it has one), the
    sum of their log-probabilities, and that sum over length ** length_penalty."""

    tokens: list[int]
    logprob: float
    score: float


class _Search:
    """The books of one prompt's search: unfinished beams (tokens, sum), best first, and finished ones."""

    def __init__(self, beams: int, end, length_penalty: float):
        self.beams, self.end, self.penalty = beams, end, length_penalty
        self.live: list[tuple[list[int], float]] = [([], 0.0)]
        self.finished: list[Hypothesis] = []

    def _hypothesis(self, tokens, total) -> Hypothesis:
        return Hypothesis(tokens, total, total / len(tokens) ** self.penalty)

    @property
    def done(self) -> bool:
        """No unfinished beam could still get ahead of the `beams` finished ones if it ended now."""
        if not self.live:
            return True
        if len(self.finished) < self.beams:
            return False
        tokens, total = self.live[0]
        return self.finished[-1].score >= total / max(1, len(tokens)) ** self.penalty

    def advance(self, totals, parents, tokens) -> list[int]:
        """Takes a selection's continuations, likeliest first (parent -1: none
        left).  Those that end are finished if they are among the first `beams`;
        the first `beams` others go on.  Returns their parents."""
        live, places = [], []
        for rank, (total, p, t) in enumerate(zip(totals, parents, tokens)):
            if p < 0 or len(live) == self.beams:
                break
            ids = self.live[p][0] + [t]
            if t == self.end:
                if rank < self.beams:
                    self.finished.append(self._hypothesis(ids, total))
            else:
                live.append((ids, total))
                places.append(p)
        self.finished.sort(key=lambda h: -h.score)  # stable: the earlier one first among equals
        del self.finished[self.beams:]
        self.live = live
        return places

    def result(self) -> list[Hypothesis]:
        """The best `beams`; unfinished ones count with the length that they have."""
        over = len(self.finished) == self.beams and self.done
        more = [] if over else [self._hypothesis(*x) for x in self.live if x[0]]
        return sorted(self.finished + more, key=lambda h: -h.score)[:self.beams]


def _host(selection):
    """A selection as lists: (totals, parents, tokens) of every group, in one copy."""
    values, parents, tokens = selection
    packed = torch.stack([values.double().view(torch.int64), parents, tokens]).cpu()
    return packed[0].view(torch.float64).tolist(), packed[1].tolist(), packed[2].tolist()


@torch.no_grad()
def generate_beams(model, prompts, beams: int, max_new_tokens: int, end_token: int | None = None,
                   length_penalty: float = 1.0, cache: PagedKVCache | None = None, page_size: int = 16,
                   graph: bool = True, dtype=torch.bfloat16) -> list[list[Hypothesis]]:
    """Beam search from prompts of different lengths (1-D int64 tensors) in one
    batch.  Returns for each prompt its best continuations (at most `beams`),
    best first by the sum of log-probabilities over length ** length_penalty.

    Every step ranks the 2 * beams likeliest continuations of a prompt's beams;
    those that end in `end_token` are finished if they are among the first
    `beams`, the first `beams` others go on.  A prompt's search ends after
    `max_new_tokens`, or when `beams` continuations are finished and none that
    goes on scores higher.  A `cache` that is passed in keeps nothing of the
    run (its pages have to suffice for every beam's own); otherwise one of `dtype` is
    made."""
    if not 1 <= beams <= 32:
        raise ValueError("1 to 32 beams")
    prompts, counts, more = check_prompts(model, prompts, max_new_tokens)
    B, K = len(prompts), beams
    if cache is None:
        unit = max(page_size, 1)  # what no page may have is for the cache to refuse
        # a prompt's full pages once, what comes behind them for every beam
        need = sum(c // unit + K * -(-(c % unit + more) // unit) for c in counts)
        cache = PagedKVCache(model.cfg, need, page_size, model.device, dtype)
    searches = [_Search(K, end_token, length_penalty) for _ in prompts]
    held: list[list[int]] = [[] for _ in prompts]  # the cache's sequences of every prompt's unfinished beams
    pads: list[int] = []
    try:
        for h in held:
            h.append(cache.add())
        ids = torch.cat([p.to(model.device) for p in prompts])
        logits = model.forward_paged(ids, cache, [h[0] for h in held], counts)
        scores = torch.zeros((B, 1), dtype=torch.float32, device=model.device)
        captured = None
        for step in range(max_new_tokens):
            totals, parents, tokens = _host(ops.beam_select(logits, scores, 2 * K))
            for g, s in enumerate(searches):
                if not s.done:
                    held[g] = cache.reorder(held[g], s.advance(totals[g], parents[g], tokens[g]))
                if s.done:
                    while held[g]:
                        cache.free(held[g].pop())
            if step + 1 == max_new_tokens or all(s.done for s in searches):
                break
            # A step always has beams times prompts places, as the graph is captured.  Where a search is over or has
            # fewer beams, an empty sequence takes the place for the step, and a score of -inf keeps it out.
            missing = B * K - sum(len(h) for h in held)
            pads += [cache.add() for _ in range(missing - len(pads))]
            spare = iter(pads)
            seqs, feed, out = [], [], []
            for h, s in zip(held, searches):
                for i in range(K):
                    tokens_so_far, total = s.live[i] if i < len(h) else ([0], -float("inf"))
                    seqs.append(h[i] if i < len(h) else next(spare))
                    feed.append(tokens_so_far[-1])
                    out.append(total)
            feed = torch.tensor(feed, dtype=torch.int64).to(model.device)
            scores = torch.tensor(out, dtype=torch.float32).view(B, K).to(model.device)
            if graph and captured is None and max_new_tokens - step > 2:
                captured = PagedDecodeGraph(model, cache, B * K, max(counts) + more, logits=True)
            logits = captured.step(seqs, feed) if captured else model.forward_paged(feed, cache, seqs)
            for q in pads:
                cache.truncate(q, 0)
    finally:
        for h in [*held, pads]:
            for q in h:
                cache.free(q)
    return [s.result() for s in searches]
