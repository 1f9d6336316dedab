"""Paged KV cache: sequences of any length in one pool of equal pages.

The contiguous caches of ``xb200.qwen`` and ``xb200.gpt2`` reserve
``[B, n_kv_head, max_seq, 64]`` per layer for a batch whose sequences all have
the same length (examples/qwen2_5/model.py:1110-1132).  Here a sequence owns
as many pages as its length needs; sequences join, fork, shrink and leave at
any time, and a step takes any of them with any number of new tokens each::

    cache = PagedKVCache(model.cfg, n_pages=4096)
    a, b = cache.add(), cache.add()
    logits = model.forward_paged(ids, cache, [a, b], [500, 37])   # two prompts, packed
    c = cache.fork(a)                                             # shares a's pages
    logits = model.forward_paged(next_ids, cache, [a, b, c])      # one token each
    cache.free(b)

The bookkeeping (who owns which page) lives on the host; the pool and the
tables that the kernels read are on the device.

With ``dtype=torch.int8`` or ``torch.float8_e4m3fn`` the pool holds codes and an
exponent byte for each position and KV head: half the bytes, so twice the
positions in the same memory and half the reading of a decode step over long
contexts.  Steps of many tokens a sequence (prompts, chunks, also beside single
tokens) expand their sequences' pages to bf16 first and take longer than over bf16
pages.  Nothing else changes for the caller.
"""

from __future__ import annotations

import heapq
from dataclasses import dataclass

import numpy as np
import torch

from . import ops


@dataclass
class PagedBatch:
    """What the paged operators read of a step: sequence b's new tokens are the
    packed rows q_start[b] .. q_start[b + 1] - 1 and its last positions."""

    page_table: torch.Tensor  # [B, columns] int32
    q_start: torch.Tensor  # [B + 1] int32
    kv_len: torch.Tensor  # [B] int32, the new tokens included
    positions: torch.Tensor  # [T] int64, of every packed token
    last: torch.Tensor | None  # [B] int64, packed row of each sequence's last token; None: one token each


def _upload(a: np.ndarray, device, out: torch.Tensor | None = None) -> torch.Tensor:
    """`a` on the device without waiting for the stream: through pinned memory
    of its own, which the host allocator reuses only after the copy has run."""
    t = torch.from_numpy(a)
    if device.type == "cuda":
        t = t.pin_memory()
    return t.to(device, non_blocking=True) if out is None else out.copy_(t, non_blocking=True)


class _Sequence:
    __slots__ = ("pages", "length")

    def __init__(self, pages, length):
        self.pages, self.length = pages, length


class PagedKVCache:
    """Pool [n_layer, 2, n_pages, n_kv_head, page_size, head_dim] (bf16, or
    int8 / float8_e4m3fn codes) and the pages of every sequence in it.

    ``k[i]`` / ``v[i]`` are layer i's pages as the operators take them, ``k_scale[i]``
    / ``v_scale[i]`` the exponents of 8-bit ones (None in bf16).  A page
    is handed out lowest number first.  Methods that move or copy pages enqueue
    the copies on the current stream, where the steps that use the cache run.
    """

    def __init__(self, cfg, n_pages: int, page_size: int = 16, device="cuda", dtype=torch.bfloat16):
        if n_pages < 1 or page_size < 8 or page_size % 8:
            raise ValueError("a pool has at least one page of a multiple of 8 positions")
        if dtype not in (torch.bfloat16, torch.int8, torch.float8_e4m3fn):
            raise ValueError("a pool holds bf16, int8 or float8_e4m3fn")
        self.n_pages, self.page_size, self.dtype = n_pages, page_size, dtype
        self.pages = torch.zeros((cfg.n_layer, 2, n_pages, cfg.n_kv_head, page_size, cfg.head_dim), dtype=dtype,
                                 device=device)
        self.k = [layer[0] for layer in self.pages]
        self.v = [layer[1] for layer in self.pages]
        self.scales = None
        self.k_scale = self.v_scale = [None] * cfg.n_layer
        if dtype is not torch.bfloat16:
            # K's and V's beside each other: a page's exponents are whole 16-byte vectors for the page copies
            self.scales = torch.zeros((cfg.n_layer, n_pages, 2, cfg.n_kv_head, page_size), dtype=torch.uint8,
                                      device=device)
            self.k_scale = [layer[:, 0] for layer in self.scales]
            self.v_scale = [layer[:, 1] for layer in self.scales]
        self.device = self.pages.device
        self._refs = [0] * n_pages
        self._free = list(range(n_pages))  # a heap
        self._seqs: dict[int, _Sequence] = {}
        self._next = 0

    # ------------------------------------------------------------- sequences

    def _get(self, seq: int) -> _Sequence:
        try:
            return self._seqs[seq]
        except KeyError:
            raise KeyError(f"no sequence {seq} in the cache") from None

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def __len__(self) -> int:
        return len(self._seqs)

    def length(self, seq: int) -> int:
        return self._get(seq).length

    def page_ids(self, seq: int) -> list[int]:
        return list(self._get(seq).pages)

    def add(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._seqs[seq] = _Sequence([], 0)
        return seq

    def fork(self, seq: int) -> int:
        """A copy of a sequence that shares its pages; a page that both still
        write into is copied when the first of them does."""
        s = self._get(seq)
        new = self.add()
        self._seqs[new] = _Sequence(list(s.pages), s.length)
        for p in s.pages:
            self._refs[p] += 1
        return new

    def _release(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    def free(self, seq: int) -> None:
        """Forget a sequence; its pages that no other one shares are free again."""
        s = self._get(seq)
        del self._seqs[seq]
        for p in s.pages:
            self._release(p)

    def truncate(self, seq: int, length: int) -> None:
        """Forget the positions from `length` on (rejected draft tokens)."""
        s = self._get(seq)
        if not 0 <= length <= s.length:
            raise ValueError(f"cannot cut a sequence of {s.length} positions at {length}")
        keep = -(-length // self.page_size)
        for p in s.pages[keep:]:
            self._release(p)
        del s.pages[keep:]
        s.length = length

    def reorder(self, seqs, parents) -> list[int]:
        """The sequences of a beam search's next step: place i goes on from
        seqs[parents[i]], which may be named several times or not at all.
        Returns the handles of the new ones; those of `seqs` that none of them
        takes over are gone."""
        seqs, parents = list(seqs), [int(p) for p in parents]
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence may appear once in a step")
        if any(not 0 <= p < len(seqs) for p in parents):
            raise ValueError(f"parents are places 0 .. {len(seqs) - 1}")
        for q in seqs:
            self._get(q)
        kept, out = set(), []
        for p in parents:  # the first to name a sequence takes it over, the others share its pages
            out.append(self.fork(seqs[p]) if p in kept else seqs[p])
            kept.add(p)
        for p, q in enumerate(seqs):
            if p not in kept:
                self.free(q)
        return out

    # ------------------------------------------------------------- steps

    def _copy(self, src, dst) -> None:
        """Pages of every layer, keys and values and their exponents."""
        ops.copy_pages(self.pages, src, dst)
        if self.scales is not None:
            ops.copy_pages(self.scales, src, dst, dim=1)

    def _grow(self, seqs, counts) -> None:
        """Room for counts[i] more positions of seqs[i], all or none: pages
        taken, and a shared page that is about to be written copied."""
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence may appear once in a step")
        if len(counts) != len(seqs) or any(c < 1 for c in counts):
            raise ValueError("every sequence of a step brings at least one token")
        P = self.page_size
        refs: dict[int, int] = {}  # changed reference counts
        plan, need = [], 0
        for q, c in zip(seqs, counts):
            s = self._get(q)
            if s.length + c > 0x7FFFFFFF:
                raise ValueError("a sequence has at most 2^31 - 1 positions")
            own = False  # whether the page that holds position s.length has to be copied
            if s.length % P:
                p = s.pages[-1]
                n = refs.get(p, self._refs[p])
                if n > 1:
                    own = True
                    refs[p] = n - 1
            fresh = -(-(s.length + c) // P) - len(s.pages)
            need += fresh + own
            plan.append((s, c, fresh, own))
        if need > len(self._free):
            raise RuntimeError(f"KV cache full: the step needs {need} pages, {len(self._free)} are free")
        taken = [heapq.heappop(self._free) for _ in range(need)]
        src, dst, at = [], [], 0
        for s, c, fresh, own in plan:
            if own:
                src.append(s.pages[-1])
                dst.append(taken[at])
            at += own + fresh
        try:  # before the books change: a copy that fails leaves them as they were
            if src:
                self._copy(src, dst)
        except BaseException:
            for p in taken:
                heapq.heappush(self._free, p)
            raise
        for p in taken:
            self._refs[p] = 1
        at = 0
        for s, c, fresh, own in plan:
            if own:
                self._refs[s.pages[-1]] -= 1
                s.pages[-1] = taken[at]
            s.pages += taken[at + own:at + own + fresh]
            at += own + fresh
            s.length += c

    def _table(self, seqs, columns: int) -> np.ndarray:
        table = np.zeros((len(seqs), columns), dtype=np.int32)
        for i, q in enumerate(seqs):
            pages = self._seqs[q].pages
            table[i, :len(pages)] = pages
        return table

    def step(self, seqs, counts=None) -> PagedBatch:
        """Takes room for counts[i] new tokens of seqs[i] (one each by
        default) and returns the batch for the operators.  Raises, with the
        cache unchanged, when the free pages do not suffice."""
        seqs = list(seqs)
        counts = [1] * len(seqs) if counts is None else [int(c) for c in counts]
        if not seqs:
            raise ValueError("a step needs at least one sequence")
        self._grow(seqs, counts)
        B = len(seqs)
        lens = np.array([self._seqs[q].length for q in seqs], dtype=np.int64)
        new = np.array(counts, dtype=np.int64)
        starts = np.zeros(B + 1, dtype=np.int64)
        np.cumsum(new, out=starts[1:])
        columns = max(len(self._seqs[q].pages) for q in seqs)
        ints = np.concatenate([self._table(seqs, columns).reshape(-1), starts, lens]).astype(np.int32)
        positions = np.arange(starts[-1]) - np.repeat(starts[1:] - lens, new)
        longs = _upload(np.concatenate([positions, starts[1:] - 1]), self.device)
        ints = _upload(ints, self.device)
        T, n = int(starts[-1]), B * columns
        return PagedBatch(ints[:n].view(B, columns), ints[n:n + B + 1], ints[n + B + 1:], longs[:T],
                          longs[T:] if T > B else None)

    def read(self, seqs, layer: int):
        """Keys and values of whole sequences in one layer, packed one after the
        other: two bf16 tensors [sum of lengths, n_kv_head, head_dim] (what
        8-bit codes stand for is a bf16 number), to hand a sequence on to
        another cache or program."""
        seqs = list(seqs)
        lens = [self._get(q).length for q in seqs]
        T, B = sum(lens), len(seqs)
        k, v = (torch.empty((T, self.pages.shape[3], self.pages.shape[5]), dtype=torch.bfloat16, device=self.device)
                for _ in range(2))
        if T:
            columns = max(len(self._seqs[q].pages) for q in seqs)
            ints = np.concatenate([self._table(seqs, columns).reshape(-1), [0], np.cumsum(lens), lens]).astype(np.int32)
            ints, n = _upload(ints, self.device), B * columns
            ops.paged_read_kv(k, v, self.k[layer], self.v[layer], ints[:n].view(B, columns), ints[n:n + B + 1],
                              ints[n + B + 1:], self.k_scale[layer], self.v_scale[layer])
        return k, v

    # ------------------------------------------------------------- the pool

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers, so that free_pages
        pages at the pool's end are unused; returns how many moved.  Batches
        and tables made before name the old places."""
        used = self.n_pages - len(self._free)
        holes = sorted(p for p in self._free if p < used)
        high = [p for p in range(used, self.n_pages) if self._refs[p]]
        assert len(holes) == len(high)
        if not high:
            return 0
        self._copy(high, holes)
        to = dict(zip(high, holes))
        for p, q in to.items():
            self._refs[q], self._refs[p] = self._refs[p], 0
        for s in self._seqs.values():
            s.pages = [to.get(p, p) for p in s.pages]
        self._free = list(range(used, self.n_pages))  # sorted: a heap
        return len(high)


def _check_cache(model, cache: PagedKVCache) -> None:
    c = model.cfg
    want, have = (c.n_layer, 2, c.n_kv_head, c.head_dim), tuple(cache.pages.shape)
    if have[:2] + have[3:4] + have[5:] != want:
        raise ValueError(f"the cache was made for another model: [n_layer, 2, n_kv_head, head_dim] is "
                         f"{have[:2] + have[3:4] + have[5:]}, the model's {want}")
    dev = model.layers[0]["qkv_w"].device
    if cache.device != dev:
        raise ValueError(f"the cache is on {cache.device}, the model on {dev}")


def check_step(model, ids, cache: PagedKVCache, seqs, counts, next_token, table: str):
    """Refuses what a step of `model` cannot take before the cache gives room
    for it; (seqs, counts) as lists.  `table` names what limits positions."""
    seqs = list(seqs)
    counts = [1] * len(seqs) if counts is None else [int(n) for n in counts]
    if ids.dim() != 1 or ids.shape[0] != sum(counts):
        raise ValueError(f"ids must be 1-D with {sum(counts)} tokens")
    for q, n in zip(seqs, counts):
        if cache.length(q) + n > model.position_limit:
            raise ValueError(f"sequence {q} would exceed the {table} ({model.position_limit})")
    _check_cache(model, cache)
    for name, t in (("ids", ids), ("next_token", next_token)):
        if t is not None and (t.dtype is not torch.int64 or t.device != cache.device):
            raise ValueError(f"{name} must be int64 on {cache.device}")
    if next_token is not None and (next_token.shape != (len(seqs),) or not next_token.is_contiguous()):
        raise ValueError(f"next_token must be contiguous [{len(seqs)}]")
    return seqs, counts


class PagedDecodeGraph:
    """One captured CUDA graph of a decode step for `batch` sequences of a
    paged cache.  The kernels read lengths and page tables from the device, so
    the same graph serves every step, whichever sequences take part and however
    long they are (up to `max_positions`).  Steps of the cache and replays run
    on one stream, or ordered by events, like any two users of the same pages.
    A step gives the greedy next tokens, or with `logits` the logits."""

    def __init__(self, model, cache: PagedKVCache, batch: int, max_positions: int, logits: bool = False):
        if batch < 1 or not 0 < max_positions <= model.position_limit:
            raise ValueError(f"batch must be positive and max_positions 1 .. {model.position_limit}")
        _check_cache(model, cache)
        self.model, self.cache, self.batch = model, cache, batch  # the graph reads the model's weights
        dev = cache.device
        self.columns = -(-max_positions // cache.page_size)
        n = batch * self.columns
        self._ints = torch.zeros(n + batch, dtype=torch.int32, device=dev)  # page table, lengths
        self.ids = torch.zeros(batch, dtype=torch.int64, device=dev)
        self.next_token = torch.zeros(batch, dtype=torch.int64, device=dev)
        self._positions = torch.zeros(batch, dtype=torch.int64, device=dev)
        # kept: the graph has the addresses of all of it
        self._step = PagedBatch(self._ints[:n].view(batch, self.columns),
                                torch.arange(batch + 1, dtype=torch.int32, device=dev), self._ints[n:],
                                self._positions, None)
        self._limit = max_positions
        # scratch buffers of this graph's own: no other call reuses or regrows them
        with ops.workspace_slot(ops.fresh_slot()):
            # one eager step of the captured sizes, a position in a page of a
            # small pool for each sequence, sets up the kernels (attributes,
            # scratch) before the capture
            small = PagedKVCache(model.cfg, batch, cache.page_size, dev, cache.dtype)
            self._step.page_table[:, 0] = torch.arange(batch, device=dev)
            self._step.kv_len.fill_(1)
            token = None if logits else self.next_token
            model.forward_packed(self.ids, small, self._step, next_token=token)
            torch.cuda.synchronize(dev)
            del small
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.logits = model.forward_packed(self.ids, cache, self._step, next_token=token)
            self._scratch = ops.take_workspace(dev)

    def step(self, seqs, ids: torch.Tensor) -> torch.Tensor:
        """The greedy next token (int64 [batch]) of every sequence after its
        token in `ids`, or the logits (fp32 [batch, vocab]); overwritten by the
        next step."""
        seqs = list(seqs)
        if len(seqs) != self.batch:
            raise ValueError(f"the graph was captured for {self.batch} sequences, got {len(seqs)}")
        if ids.shape != self.ids.shape or ids.dtype is not torch.int64:
            raise ValueError(f"ids must be int64 [{self.batch}]")
        if any(self.cache.length(q) >= self._limit for q in seqs):
            raise ValueError(f"a sequence would outgrow the graph's {self._limit} positions")
        self.cache._grow(seqs, [1] * len(seqs))
        lens = np.array([self.cache.length(q) for q in seqs], dtype=np.int64)
        ints = np.concatenate([self.cache._table(seqs, self.columns).reshape(-1), lens]).astype(np.int32)
        _upload(ints, self.cache.device, self._ints)
        _upload(lens - 1, self.cache.device, self._positions)
        self.ids.copy_(ids)
        self.graph.replay()
        return self.next_token if self.logits is None else self.logits


def check_prompts(model, prompts, max_new_tokens: int):
    """(prompts, their lengths, positions behind them: the last token is never fed back)"""
    prompts = list(prompts)
    if not prompts or any(p.dim() != 1 or p.numel() == 0 for p in prompts) or max_new_tokens < 1:
        raise ValueError("prompts are non-empty 1-D tensors, and at least one token is generated")
    counts = [p.numel() for p in prompts]
    more = max_new_tokens - 1
    if max(counts) + more > model.position_limit:
        raise ValueError(f"{max(counts) + more} positions exceed the model's {model.position_limit}")
    return prompts, counts, more


def generate_paged(model, prompts, max_new_tokens: int, cache: PagedKVCache | None = None, page_size: int = 16,
                   graph: bool = True, dtype=torch.bfloat16) -> torch.Tensor:
    """Greedy continuation of prompts of different lengths (1-D int64 tensors)
    in one batch: the prompts are prefilled packed, then every sequence decodes
    a token per step.  Returns tokens [B, max_new_tokens] on the device; a
    `cache` that is passed in keeps nothing of the run, otherwise one of `dtype`
    is made for it."""
    prompts, counts, more = check_prompts(model, prompts, max_new_tokens)
    longest = max(counts) + more
    if cache is None:
        unit = max(page_size, 1)  # what no page may have is for the cache to refuse
        cache = PagedKVCache(model.cfg, sum(-(-(c + more) // unit) for c in counts), page_size, model.device, dtype)
    B = len(prompts)
    ids = torch.cat([p.to(model.device) for p in prompts])
    toks = torch.empty((max_new_tokens, B), dtype=torch.int64, device=model.device)
    seqs = [cache.add() for _ in prompts]
    try:
        model.forward_paged(ids, cache, seqs, counts, next_token=toks[0])
        if graph and max_new_tokens > 2:
            g = PagedDecodeGraph(model, cache, B, longest)
            for i in range(1, max_new_tokens):
                toks[i].copy_(g.step(seqs, toks[i - 1]))
        else:
            for i in range(1, max_new_tokens):
                model.forward_paged(toks[i - 1], cache, seqs, next_token=toks[i])
    finally:
        for q in seqs:
            cache.free(q)
    return toks.t()
