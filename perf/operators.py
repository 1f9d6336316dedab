"""The operators of a paged KV cache: what they compute, on which sizes, in plain torch and on the xb200 kernels.

A paged cache keeps the keys and values of many sequences in one pool of
equal pages; a page table lists each sequence's pages in order.  A step of a
model brings some new tokens of every sequence (one when it decodes, many for
a prompt or a chunk of one), packed without padding: tokens
``q_start[b] .. q_start[b + 1] - 1`` are the last ones of sequence b, which
with them holds ``kv_len[b]`` positions.

``rope``       rotate the new queries and keys to their positions (none for
               learned positions) and write keys and values into the pages;
``attention``  causal grouped-query attention of the new tokens over the pages;
``copy``       copy pages within the pool, all layers at once: the page that a
               forked sequence may not share, or the moves of a compaction.

``own`` selects the xb200 kernels; otherwise ``run`` computes the same in
elementary torch operations in 32 bits, rounded once at the end.
"""

import math
import os
import random
import sys

import torch

own = False

HEAD_DIM = 64  # of every attention in this repository
LAYERS = {2: 24, 12: 12}  # decoder layers of the models with 2 and with 12 KV heads; others: 8


# ----------------------------------------------------------------------------- cases


def listed():
    return [
        # one user's chat: a single token over a short context, where latency is all
        dict(name="decode 1 seq", op="attention", batch=1, heads=14, kv_heads=2, page=16, chunks=0, chunk_lo=1,
             chunk_hi=1, past_lo=511, past_hi=511, lens=1),
        # the batch of the repository's own generation benchmark (64 x 512 + 128 tokens), lengths ragged
        dict(name="decode 64 seqs", op="attention", batch=64, heads=14, kv_heads=2, page=16, chunks=0, chunk_lo=1,
             chunk_hi=1, past_lo=512, past_hi=639, lens=2),
        # a full server: many sequences from short to very long
        dict(name="decode 160 long seqs", op="attention", batch=160, heads=14, kv_heads=2, page=64, chunks=0,
             chunk_lo=1, chunk_hi=1, past_lo=200, past_hi=30000, lens=3),
        # the same for multi-head attention, one query head per KV head
        dict(name="decode 100 seqs mha", op="attention", batch=100, heads=12, kv_heads=12, page=32, chunks=0,
             chunk_lo=1, chunk_hi=1, past_lo=100, past_hi=1023, lens=4),
        # drafted tokens verified together: a few tokens of each sequence
        dict(name="verify 5 tokens", op="attention", batch=33, heads=14, kv_heads=2, page=16, chunks=33, chunk_lo=5,
             chunk_hi=5, past_lo=300, past_hi=4000, lens=5),
        # prompts of different lengths prefilled in one batch
        dict(name="prompts", op="attention", batch=24, heads=14, kv_heads=2, page=16, chunks=24, chunk_lo=130,
             chunk_hi=1021, past_lo=0, past_hi=0, lens=6),
        # decoding sequences share the step with chunks of long prompts
        dict(name="decode with chunks", op="attention", batch=50, heads=14, kv_heads=2, page=16, chunks=3,
             chunk_lo=480, chunk_hi=512, past_lo=100, past_hi=4000, lens=7),
        # the last chunk of a 32768-token prompt
        dict(name="chunk at 28672", op="attention", batch=1, heads=14, kv_heads=2, page=64, chunks=1, chunk_lo=4096,
             chunk_hi=4096, past_lo=28672, past_hi=28672, lens=8),
        # a decode step's keys and values
        dict(name="rope decode", op="rope", batch=64, heads=14, kv_heads=2, page=16, chunks=0, chunk_lo=1, chunk_hi=1,
             past_lo=512, past_hi=639, rotate=True, lens=9),
        # a prefill's
        dict(name="rope prefill", op="rope", batch=61, heads=14, kv_heads=2, page=16, chunks=61, chunk_lo=300,
             chunk_hi=900, past_lo=0, past_hi=500, rotate=True, lens=10),
        # four sequences forked: the partly filled last page of each
        dict(name="fork 4 seqs", op="copy", kv_heads=2, page=16, copies=4, pool=2000),
        # a fragmented pool compacted
        dict(name="compact 2500 pages", op="copy", kv_heads=2, page=16, copies=2500, pool=8000),
    ]


HEADS = [(14, 2), (12, 12), (16, 16), (16, 4), (20, 4), (8, 1), (10, 2), (9, 3), (16, 1), (25, 25), (32, 8)]


def draw(rng):
    """One more case: any operator, head layout and page size, one token to whole prompts, short to long contexts."""
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["attention", "attention", "attention", "rope", "copy"])
    heads, kv_heads = rng.choice(HEADS)
    page = rng.choice([8, 16, 16, 32, 48, 64, 128])
    if op == "copy":
        copies = log(1, 2500)
        case = dict(op=op, kv_heads=kv_heads, page=page, copies=copies, pool=2 * copies + rng.randrange(1, 3000))
        while work(case)["bytes"] > 9e8 or _pool_bytes(case) > 6e9:
            case["copies"] = case["copies"] // 2 + 1
            case["pool"] = case["pool"] // 2 + 2
        return case
    case = dict(op=op, batch=log(1, 200), heads=heads, kv_heads=kv_heads, page=page, lens=rng.randrange(1 << 30))
    kind = rng.choice(["decode", "few", "prompts", "mixed"])
    lo = log(1, 400)
    case["chunks"] = 0 if kind == "decode" else rng.randrange(0, case["batch"] + 1) if kind == "mixed" else case["batch"]
    case["chunk_lo"] = lo if kind in ("prompts", "mixed") else rng.randrange(1, 5)
    case["chunk_hi"] = case["chunk_lo"] + (log(1, 1600) if kind in ("prompts", "mixed") else rng.randrange(0, 8))
    case["past_lo"] = 0 if rng.random() < 0.3 else log(1, 2000)
    case["past_hi"] = case["past_lo"] + (0 if rng.random() < 0.1 else log(1, 20000))
    if op == "rope":
        case["rotate"] = rng.random() < 0.8
    largest = listed()[7]
    while True:
        w, top = work(case), work(largest)
        n, past = _lengths(case)
        scores = len(n) * heads * max(n) * max(a + b for a, b in zip(n, past))  # what the plain form holds at once
        keys = len(n) * kv_heads * max(a + b for a, b in zip(n, past)) * HEAD_DIM
        if w["flops"] <= top["flops"] and w["bytes"] <= 5e8 and scores <= 1.5e9 and keys <= 1.5e9:
            return case
        case["batch"] = (case["batch"] + 1) // 2
        case["chunks"] = (case["chunks"] + 1) // 2
        case["chunk_hi"] = max(case["chunk_lo"], case["chunk_hi"] * 3 // 4)
        case["past_hi"] = max(case["past_lo"], case["past_hi"] * 3 // 4)


def _lengths(case):
    """(new tokens, tokens before them) of every sequence: the case's own, whatever the inputs' seed."""
    rng = random.Random(case["lens"])
    chunked = set(rng.sample(range(case["batch"]), case["chunks"]))
    new = [rng.randint(case["chunk_lo"], case["chunk_hi"]) if b in chunked else 1 for b in range(case["batch"])]
    lo, hi = case["past_lo"] + 1, case["past_hi"] + 1
    past = [min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))) - 1 for _ in range(case["batch"])]
    return new, past


def _pool_bytes(case):
    return LAYERS.get(case["kv_heads"], 8) * 2 * case["pool"] * case["kv_heads"] * case["page"] * HEAD_DIM * 2


# ----------------------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = random.Random(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)

    D, KVH, P = HEAD_DIM, case["kv_heads"], case["page"]
    if case["op"] == "copy":
        L, n, c = LAYERS.get(KVH, 8), case["pool"], case["copies"]
        pages = torch.empty((L, 2, n, KVH, P, D), dtype=torch.bfloat16, device="cuda")
        for layer in pages:  # by layers: the 32-bit numbers behind a whole pool would fill the card
            layer.copy_(normal(2, n, KVH, P, D))
        ids = order.sample(range(n), 2 * c)
        return dict(op="copy", pages=pages, src=torch.tensor(ids[:c], dtype=torch.int32),
                    dst=torch.tensor(ids[c:], dtype=torch.int32))

    H, B = case["heads"], case["batch"]
    new, past = _lengths(case)
    length = [a + b for a, b in zip(new, past)]
    used = [-(-x // P) for x in length]
    n_pages = sum(used) + max(4, sum(used) // 8)
    free = list(range(n_pages))  # pages in the order a pool hands them out after some churn
    order.shuffle(free)
    table = torch.zeros((B, max(used)), dtype=torch.int32)
    for b, u in enumerate(used):
        table[b, :u] = torch.tensor(free[:u], dtype=torch.int32)
        del free[:u]
    T = sum(new)
    starts = [0]
    for x in new:
        starts.append(starts[-1] + x)
    state = dict(op=case["op"], heads=H, kv_heads=KVH, page=P, max_new=max(new), max_len=max(length),
                 q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 kv_len=torch.tensor(length, dtype=torch.int32, device="cuda"), page_table=table.cuda(),
                 k_pages=normal(n_pages, KVH, P, D), v_pages=normal(n_pages, KVH, P, D))
    if case["op"] == "attention":
        return dict(state, q=normal(T, H, D, scale=2.0), scale=1.0 / math.sqrt(D),
                    out=torch.zeros((T, H * D), dtype=torch.bfloat16, device="cuda"))
    cos = sin = None
    if case["rotate"]:
        freq = 1e6 ** (-torch.arange(D // 2, dtype=torch.float64, device="cuda") / (D // 2))
        angle = torch.outer(torch.arange(max(length), dtype=torch.float64, device="cuda"), freq).repeat(1, 2)
        cos, sin = angle.cos().float(), angle.sin().float()
    return dict(state, qkv=normal(T, (H + 2 * KVH) * D), cos=cos, sin=sin,
                q=torch.zeros((T, H, D), dtype=torch.bfloat16, device="cuda"))


# ----------------------------------------------------------------------------- one pass


def run(state):
    s = state
    if own:
        try:
            from xb200 import ops
        except ModuleNotFoundError:  # the package's folder is no package name: put on the path, as bench.py does
            sys.path.insert(0, os.path.join(os.getcwd(), "triton-xdna_b200"))
            from xb200 import ops

        if s["op"] == "copy":
            return ops.copy_pages(s["pages"], s["src"], s["dst"])
        if s["op"] == "rope":
            ops.paged_rope_kv(s["qkv"], s["cos"], s["sin"], s["q"], s["k_pages"], s["v_pages"], s["page_table"],
                              s["q_start"], s["kv_len"])
            return s["q"], s["k_pages"], s["v_pages"]
        return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["out"], s["page_table"], s["q_start"],
                                   s["kv_len"], s["scale"])
    if s["op"] == "copy":
        src, dst = s["src"].cuda(), s["dst"].cuda()
        s["pages"][:, :, dst] = s["pages"][:, :, src]
        return s["pages"]
    return _plain_rope(s) if s["op"] == "rope" else _plain_attention(s)


def _positions(s, tokens):
    """The sequence and the position of every packed token."""
    t = torch.arange(tokens, device="cuda")
    seq = (t[:, None] >= s["q_start"][None, 1:]).sum(1)
    return seq, s["kv_len"][seq] - s["q_start"][seq + 1] + t


def _plain_rope(s):
    H, KVH, D = s["heads"], s["kv_heads"], HEAD_DIM
    x = s["qkv"].float().view(-1, H + 2 * KVH, D)
    seq, pos = _positions(s, x.shape[0])
    qk, v = x[:, :H + KVH], x[:, H + KVH:]
    if s["cos"] is not None:
        cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
        qk = qk * cos + torch.cat([-qk[..., D // 2:], qk[..., :D // 2]], -1) * sin
    s["q"].copy_(qk[:, :H])
    page, row = s["page_table"][seq, pos // s["page"]].long(), pos % s["page"]
    s["k_pages"][page, :, row] = qk[:, H:].to(torch.bfloat16)
    s["v_pages"][page, :, row] = v.to(torch.bfloat16)
    return s["q"], s["k_pages"], s["v_pages"]


def _plain_attention(s):
    H, KVH, D = s["heads"], s["kv_heads"], HEAD_DIM
    T, B, N, L = s["q"].shape[0], s["kv_len"].shape[0], s["max_new"], s["max_len"]
    first, count = s["q_start"][:-1], s["q_start"][1:] - s["q_start"][:-1]
    at = torch.arange(N, device="cuda")
    q = s["q"][(first[:, None] + at).clamp(max=T - 1)].float()  # [B, N, H, D], padded to the longest chunk
    q = q.view(B, N, KVH, H // KVH, D).permute(0, 2, 3, 1, 4).reshape(B, KVH, H // KVH * N, D)
    key = torch.arange(L, device="cuda")
    page, row = s["page_table"][:, key // s["page"]].long(), key % s["page"]
    held = key < s["kv_len"][:, None]  # [B, L]: behind it lies whatever the page held before
    k = s["k_pages"][page, :, row].float().transpose(1, 2)  # [B, KVH, L, D]
    v = torch.where(held[:, :, None, None], s["v_pages"][page, :, row].float(), 0.0).transpose(1, 2)
    score = (q @ k.transpose(-1, -2)).view(B, KVH, H // KVH, N, L) * s["scale"]
    seen = key <= (s["kv_len"] - count)[:, None, None] + at[:, None]  # [B, N, L]
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, KVH, H // KVH * N, L) @ v).view(B, KVH, H // KVH, N, D) / torch.where(total > 0, total, 1.0)
    t = torch.arange(T, device="cuda")
    seq = (t[:, None] >= s["q_start"][None, 1:]).sum(1)
    s["out"].copy_(o[seq, :, :, t - first[seq]].reshape(T, H * D))
    return s["out"]


# ----------------------------------------------------------------------------- what it takes


def work(case):
    D, KVH = HEAD_DIM, case["kv_heads"]
    if case["op"] == "copy":
        return {"bytes": 2 * LAYERS.get(KVH, 8) * 2 * case["copies"] * KVH * case["page"] * D * 2, "flops": 0}
    H = case["heads"]
    new, past = _lengths(case)
    T = sum(new)
    index = 4 * (2 * len(new) + 1 + sum(-(-(a + b) // case["page"]) for a, b in zip(new, past)))
    if case["op"] == "rope":  # packed rows in; queries, keys and values out; the table rows of the positions
        table = 2 * 4 * D * T if case["rotate"] else 0
        flops = 3 * T * (H + KVH) * D if case["rotate"] else 0
        return {"bytes": 2 * 2 * T * (H + 2 * KVH) * D + min(table, 2 * 4 * D * 32768) + index, "flops": flops}
    keys = sum(a + b for a, b in zip(new, past))
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, past))  # (token, key it sees)
    return {"bytes": 2 * 2 * keys * KVH * D + 2 * 2 * T * H * D + index, "flops": 4 * pairs * H * D}


# ----------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    """What run() returns, sequence by sequence and head by head from the definitions, in 64 bits."""
    s = prepare(case, seed)
    if s["op"] == "copy":
        was = s["pages"].clone()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            s["pages"][:, :, b] = was[:, :, a]
        return s["pages"]
    new, past = _lengths(case)
    P, H, KVH, D = case["page"], case["heads"], case["kv_heads"], HEAD_DIM
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    if s["op"] == "rope":
        q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        t = 0
        for b, (n, before) in enumerate(zip(new, past)):
            pages = s["page_table"][b].tolist()
            rows = s["qkv"][t:t + n].double().view(n, H + 2 * KVH, D)
            z = torch.complex(rows[..., :D // 2].contiguous(), rows[..., D // 2:].contiguous())
            if case["rotate"]:
                turn = torch.complex(s["cos"][before:before + n, :D // 2].double(),
                                     s["sin"][before:before + n, :D // 2].double())
                z = z * turn[:, None]
            turned = torch.cat([z.real, z.imag], -1)
            q[t:t + n] = turned[:, :H]
            i = 0
            while i < n:  # page by page
                at, row = pages[(before + i) // P], (before + i) % P
                c = min(P - row, n - i)
                k_pages[at, :, row:row + c] = turned[i:i + c, H:H + KVH].transpose(0, 1)
                v_pages[at, :, row:row + c] = rows[i:i + c, H + KVH:].transpose(0, 1)
                i += c
            t += n
        return q, k_pages, v_pages
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    t = 0
    for b, (n, before) in enumerate(zip(new, past)):
        pages = s["page_table"][b, :-(-(n + before) // P)].long()
        hidden = torch.ones((n, n + before), dtype=torch.bool, device="cuda").triu(before + 1)
        for h in range(H):
            k = k_pages[pages, h // (H // KVH)].reshape(-1, D)[:n + before]
            v = v_pages[pages, h // (H // KVH)].reshape(-1, D)[:n + before]
            score = (s["q"][t:t + n, h].double() @ k.T * s["scale"]).masked_fill_(hidden, -math.inf)
            out[t:t + n, h * D:(h + 1) * D] = torch.softmax(score, -1) @ v
        t += n
    return out
