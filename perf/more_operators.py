"""Operators of an 8-bit paged KV cache and of beam search over it: what they compute, on which sizes, in plain torch and on the xb200 kernels.

An 8-bit paged cache holds keys and values as int8 or float8_e4m3fn codes in
the pages that ``perf/operators.py`` describes (packed new tokens, page tables,
``q_start`` and ``kv_len``), with one exponent byte for each position and KV
head: a code c stands for c * 2^(byte - 127), and byte 255 makes its whole vector
NaN.  The exponent of a vector is the smallest that keeps its largest
magnitude within the codes' range (127 or 448), so what a code stands for is
always a bf16 number.

``attention``  causal grouped-query attention of the packed new tokens over the pages;
``write``      rotate the new queries and keys to their positions, write keys and values into the pages as
               codes, and read them back;
``read``       the keys and values of whole sequences, out of their pages, as bf16;
``beam``       the best continuations of each group's beams over the vocabulary: the sums of a beam's score
               and a token's log-probability, largest first, equal ones by the lowest (beam, token).

``own`` selects the xb200 kernels; otherwise ``run`` computes the same in
elementary torch operations.
"""

import math
import random

import torch

own = False

HEAD_DIM = 64  # of every attention in this repository
CODES = {"int8": (torch.int8, 127.0, 6, 126, 248), "fp8": (torch.float8_e4m3fn, 448.0, 8, 96, 246)}
LEAST = 47  # smallest exponent byte


# ----------------------------------------------------------------------------- cases


def listed():
    return [
        # one user's chat: a single token over a short context, where latency is all
        dict(name="decode 1 seq int8", op="attention", code="int8", batch=1, heads=14, kv_heads=2, page=16, chunks=0,
             chunk_lo=1, chunk_hi=1, past_lo=511, past_hi=511, share=1, lens=1),
        # the batch of the repository's own generation benchmark (64 x 512 + 128 tokens), lengths ragged
        dict(name="decode 64 seqs fp8", op="attention", code="fp8", batch=64, heads=14, kv_heads=2, page=16, chunks=0,
             chunk_lo=1, chunk_hi=1, past_lo=512, past_hi=639, share=1, lens=2),
        # a full server: many sequences from short to very long
        dict(name="decode 160 long seqs int8", op="attention", code="int8", batch=160, heads=14, kv_heads=2, page=64,
             chunks=0, chunk_lo=1, chunk_hi=1, past_lo=200, past_hi=30000, share=1, lens=3),
        # 25 searches of four beams, which share the pages of their prompts; one query head per KV head
        dict(name="decode 25 x 4 beams fp8", op="attention", code="fp8", batch=100, heads=12, kv_heads=12, page=32,
             chunks=0, chunk_lo=1, chunk_hi=1, past_lo=100, past_hi=1023, share=4, lens=4),
        # prompts of different lengths prefilled in one batch
        dict(name="prompts int8", op="attention", code="int8", batch=24, heads=14, kv_heads=2, page=16, chunks=24,
             chunk_lo=130, chunk_hi=1021, past_lo=0, past_hi=0, share=1, lens=6),
        # the last chunk of a 32768-token prompt
        dict(name="chunk at 28672 fp8", op="attention", code="fp8", batch=1, heads=14, kv_heads=2, page=64, chunks=1,
             chunk_lo=4096, chunk_hi=4096, past_lo=28672, past_hi=28672, share=1, lens=8),
        # a decode step's keys and values
        dict(name="write decode int8", op="write", code="int8", batch=64, heads=14, kv_heads=2, page=16, chunks=0,
             chunk_lo=1, chunk_hi=1, past_lo=512, past_hi=639, share=1, rotate=True, lens=9),
        # a prefill's
        dict(name="write prefill fp8", op="write", code="fp8", batch=61, heads=14, kv_heads=2, page=16, chunks=61,
             chunk_lo=300, chunk_hi=900, past_lo=0, past_hi=500, share=1, rotate=True, lens=10),
        # a batch of sequences handed on to a cache in bf16
        dict(name="read 40 seqs int8", op="read", code="int8", batch=40, heads=14, kv_heads=2, page=16, chunks=0,
             chunk_lo=1, chunk_hi=1, past_lo=300, past_hi=8000, share=1, lens=11),
        # one search of four beams over the larger of the repository's vocabularies
        dict(name="beam 1 x 4", op="beam", dtype="float32", groups=1, beams=4, vocab=151936, pitch=151936, count=8,
             banned=0, first=False),
        # a batch of searches of eight beams
        dict(name="beam 32 x 8", op="beam", dtype="float32", groups=32, beams=8, vocab=151936, pitch=151936, count=16,
             banned=20, first=False),
        # the smaller vocabulary, odd, in bf16 (many equal logits), out of padded rows
        dict(name="beam 48 x 5 bf16", op="beam", dtype="bfloat16", groups=48, beams=5, vocab=50257, pitch=50304,
             count=10, banned=3, first=False),
    ]


HEADS = [(14, 2), (12, 12), (16, 16), (16, 4), (20, 4), (8, 1), (10, 2), (9, 3), (16, 1), (25, 25), (32, 8)]


def draw(rng):
    """One more case: any operator, code, head layout and page size, one token to whole prompts, short to long contexts;
    any number of searches and beams, small to large vocabularies."""
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["attention", "attention", "attention", "write", "read", "beam", "beam"])
    if op == "beam":
        groups, beams, vocab = log(1, 64), rng.randrange(1, 17), log(1000, 152000)
        while groups * beams * vocab > 32 * 8 * 151936:
            groups = (groups + 1) // 2
        return dict(op=op, dtype=rng.choice(["float32", "float32", "bfloat16"]), groups=groups, beams=beams, vocab=vocab,
                    pitch=vocab + rng.choice([0, 0, rng.randrange(1, 200)]), count=beams * rng.choice([1, 2, 2]),
                    banned=rng.choice([0, log(1, 500)]), first=rng.random() < 0.2)
    heads, kv_heads = rng.choice(HEADS)
    case = dict(op=op, code=rng.choice(["int8", "fp8"]), batch=log(1, 200), heads=heads, kv_heads=kv_heads,
                page=rng.choice([8, 16, 16, 32, 48, 64, 128]), lens=rng.randrange(1 << 30))
    kind = "decode" if op == "read" else rng.choice(["decode", "few", "prompts", "mixed"])
    lo = log(1, 400)
    case["chunks"] = 0 if kind == "decode" else rng.randrange(0, case["batch"] + 1) if kind == "mixed" else case["batch"]
    case["chunk_lo"] = lo if kind in ("prompts", "mixed") else rng.randrange(1, 5)
    case["chunk_hi"] = case["chunk_lo"] + (log(1, 1600) if kind in ("prompts", "mixed") else rng.randrange(0, 8))
    case["past_lo"] = 0 if rng.random() < 0.3 else log(1, 2000)
    case["past_hi"] = case["past_lo"] + (0 if rng.random() < 0.1 else log(1, 20000))
    case["share"] = rng.choice([2, 4, 5]) if kind == "decode" and op == "attention" and rng.random() < 0.3 else 1
    if op == "write":
        case["rotate"] = rng.random() < 0.8
    top = work(listed()[5])["flops"]
    while True:
        w = work(case)
        n, past = _lengths(case)
        scores = len(n) * heads * max(n) * max(a + b for a, b in zip(n, past))  # what the plain form holds at once
        keys = len(n) * kv_heads * max(a + b for a, b in zip(n, past)) * HEAD_DIM
        if w["flops"] <= top and w["bytes"] <= 4e8 and scores <= 1.5e9 and keys <= 1.5e9:
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
    for b in range(case["batch"]):  # the beams of one search are equally long
        past[b] = past[b - b % case["share"]]
    return new, past


# ----------------------------------------------------------------------------- codes


def _quantise(x, code):
    """Codes and exponent bytes of the vectors x [..., D] of bf16 numbers (in 32 bits)."""
    dtype, most, bits, fraction, last = CODES[code]
    top = x.abs().amax(-1).view(torch.int32)  # the bits of a number that is not negative
    byte = ((top >> 23) - bits + ((top >> 16 & 127) > fraction).int()).clamp(LEAST, last)
    bad = top >= 0x7F800000  # infinity or NaN
    step = ((254 - byte) << 23).view(torch.float32)[..., None]  # 2^-e
    y = torch.where(bad[..., None], 0.0, (x * step)).clamp(-most, most)
    return (y.round() if code == "int8" else y).to(dtype), torch.where(bad, 255, byte).to(torch.uint8)


def _values(codes, bytes_):
    """What they stand for, in 32 bits."""
    e = bytes_.int()
    return codes.float() * torch.where(e == 255, 0x7FC00000, e << 23).view(torch.float32)[..., None]


# ----------------------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "beam":
        return _prepare_beam(case, g)
    order = random.Random(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)

    D, KVH, P = HEAD_DIM, case["kv_heads"], case["page"]
    H, B = case["heads"], case["batch"]
    new, past = _lengths(case)
    length = [a + b for a, b in zip(new, past)]
    used = [-(-x // P) for x in length]
    n_pages = sum(used) + max(4, sum(used) // 8)
    free = list(range(n_pages))  # pages in the order a pool hands them out after some churn
    order.shuffle(free)
    table = torch.zeros((B, max(used)), dtype=torch.int32)
    for b, u in enumerate(used):
        own_from = 0 if b % case["share"] == 0 else past[b] // P  # full pages of the search's prompt are shared
        table[b, :own_from] = table[b - b % case["share"], :own_from]
        table[b, own_from:u] = torch.tensor(free[:u - own_from], dtype=torch.int32)
        del free[:u - own_from]
    T = sum(new)
    starts = [0]
    for x in new:
        starts.append(starts[-1] + x)

    def pages():
        """A pool of codes: keys or values whose size varies from token to token, with a few large channels."""
        codes = torch.empty((n_pages, KVH, P, D), dtype=CODES[case["code"]][0], device="cuda")
        bytes_ = torch.empty((n_pages, KVH, P), dtype=torch.uint8, device="cuda")
        channel = 1.0 + 3.0 * (torch.rand((KVH, 1, D), generator=g, device="cuda") > 0.95)
        for i in range(0, n_pages, 8192):  # by parts: the 32-bit numbers behind a whole pool would fill the card
            n = min(8192, n_pages - i)
            size = torch.exp(0.4 * torch.randn((n, KVH, P, 1), generator=g, device="cuda"))
            x = (torch.randn((n, KVH, P, D), generator=g, device="cuda") * size * channel).to(torch.bfloat16).float()
            codes[i:i + n], bytes_[i:i + n] = _quantise(x, case["code"])
        return codes, bytes_

    k_pages, k_scale = pages()
    v_pages, v_scale = pages()
    state = dict(op=case["op"], code=case["code"], heads=H, kv_heads=KVH, page=P, max_new=max(new), max_len=max(length),
                 q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 kv_len=torch.tensor(length, dtype=torch.int32, device="cuda"), page_table=table.cuda(),
                 k_pages=k_pages, v_pages=v_pages, k_scale=k_scale, v_scale=v_scale)
    if case["op"] == "attention":
        return dict(state, q=normal(T, H, D, scale=1.5), scale=1.0 / math.sqrt(D),
                    out=torch.zeros((T, H * D), dtype=torch.bfloat16, device="cuda"))

    def empty(rows):
        return torch.zeros((rows, KVH, D), dtype=torch.bfloat16, device="cuda")

    if case["op"] == "read":  # whole sequences: every position is one to read
        ends = torch.tensor([0] + length, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
        return dict(state, q_start=ends, k_out=empty(sum(length)), v_out=empty(sum(length)))
    cos = sin = None
    if case["rotate"]:
        freq = 1e6 ** (-torch.arange(D // 2, dtype=torch.float64, device="cuda") / (D // 2))
        angle = torch.outer(torch.arange(max(length), dtype=torch.float64, device="cuda"), freq).repeat(1, 2)
        cos, sin = angle.cos().float(), angle.sin().float()
    return dict(state, qkv=normal(T, (H + 2 * KVH) * D), cos=cos, sin=sin, k_out=empty(T), v_out=empty(T),
                q=torch.zeros((T, H, D), dtype=torch.bfloat16, device="cuda"))


def _prepare_beam(case, g):
    R, V, dtype = case["groups"] * case["beams"], case["vocab"], getattr(torch, case["dtype"])
    logits = torch.empty((R, case["pitch"]), dtype=dtype, device="cuda")
    # a few likely tokens stand out of many unlikely ones
    logits.copy_(2.0 * torch.randn(logits.shape, generator=g, device="cuda"))
    likely = torch.randint(0, V // 12, (R, 12), generator=g, device="cuda") + torch.arange(12, device="cuda") * (V // 12)
    logits.scatter_add_(1, likely, (4.0 + 5.0 * torch.rand(likely.shape, generator=g, device="cuda")).to(dtype))
    if case["banned"]:
        logits[:, torch.randint(0, V, (case["banned"],), generator=g, device="cuda")] = -math.inf
    scores = -20.0 + 2.0 * torch.randn((case["groups"], case["beams"]), generator=g, device="cuda")
    scores = scores.sort(1, descending=True).values
    if case["first"]:  # of the first step's beams, which are all alike, one counts
        scores[:, 0], scores[:, 1:] = 0.0, -math.inf
    return dict(op="beam", logits=logits[:, :V], scores=scores, count=case["count"])


# ----------------------------------------------------------------------------- one pass


def run(state):
    s = state
    if own:
        from xb200 import ops

        if s["op"] == "beam":
            return ops.beam_select(s["logits"], s["scores"], s["count"])
        pages = (s["k_pages"], s["v_pages"])
        at = (s["page_table"], s["q_start"], s["kv_len"])
        if s["op"] == "attention":
            return ops.paged_attention(s["q"], *pages, s["out"], *at, s["scale"], s["k_scale"], s["v_scale"])
        if s["op"] == "write":
            ops.paged_rope_kv(s["qkv"], s["cos"], s["sin"], s["q"], *pages, *at, s["k_scale"], s["v_scale"])
        ops.paged_read_kv(s["k_out"], s["v_out"], *pages, *at, s["k_scale"], s["v_scale"])
        return (s["q"], s["k_out"], s["v_out"]) if s["op"] == "write" else (s["k_out"], s["v_out"])
    return {"beam": _plain_beam, "attention": _plain_attention, "write": _plain_write, "read": _plain_read}[s["op"]](s)


def _positions(s, tokens):
    """The page, the row in it and the position of every packed token."""
    t = torch.arange(tokens, device="cuda")
    seq = (t[:, None] >= s["q_start"][None, 1:]).sum(1)
    pos = s["kv_len"][seq] - s["q_start"][seq + 1] + t
    return s["page_table"][seq, pos // s["page"]].long(), pos % s["page"], pos


def _plain_write(s):
    H, KVH, D = s["heads"], s["kv_heads"], HEAD_DIM
    x = s["qkv"].float().view(-1, H + 2 * KVH, D)
    page, row, pos = _positions(s, x.shape[0])
    qk, v = x[:, :H + KVH], x[:, H + KVH:]
    if s["cos"] is not None:
        cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
        qk = qk * cos + torch.cat([-qk[..., D // 2:], qk[..., :D // 2]], -1) * sin
    qk = qk.to(torch.bfloat16)  # what a cache in bf16 holds is what is quantised
    s["q"].copy_(qk[:, :H])
    s["k_pages"][page, :, row], s["k_scale"][page, :, row] = _quantise(qk[:, H:].float(), s["code"])
    s["v_pages"][page, :, row], s["v_scale"][page, :, row] = _quantise(v, s["code"])
    return s["q"], *_plain_read(s)


def _plain_read(s):
    page, row, _ = _positions(s, s["k_out"].shape[0])
    s["k_out"].copy_(_values(s["k_pages"][page, :, row], s["k_scale"][page, :, row]))
    s["v_out"].copy_(_values(s["v_pages"][page, :, row], s["v_scale"][page, :, row]))
    return s["k_out"], s["v_out"]


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
    k = _values(s["k_pages"][page, :, row], s["k_scale"][page, :, row]).transpose(1, 2)  # [B, KVH, L, D]
    v = _values(s["v_pages"][page, :, row], s["v_scale"][page, :, row])
    v = torch.where(held[:, :, None, None], v, 0.0).transpose(1, 2)
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


def _plain_beam(s):
    (G, K), (R, V), N = s["scores"].shape, s["logits"].shape, s["count"]
    x = s["logits"].float()
    # 64 bits from here on: sums of two beams may lie closer than 32 tell apart
    top = x.amax(1, keepdim=True).double()
    lse = top + torch.log(torch.exp(x.double() - top).sum(1, keepdim=True))
    # a row's best logits, the lower token first where two are equal: one whole number that orders both
    bits = torch.where(x == 0, 0.0, x).view(torch.int32).long()
    order = torch.where(bits < 0, -0x80000000 - bits, bits) * V + (V - 1 - torch.arange(V, device=x.device))
    n = min(N, V)
    token = V - 1 - order.topk(n, 1).values.sort(1, descending=True).values % V  # [R, n]
    total = s["scores"].double().view(R, 1) + x.gather(1, token).double() - lse
    total = torch.where(total.isfinite(), total, -math.inf).view(G, K, n)
    # the beams' lists joined: rank of each by the sums, equal ones in (beam, token) order, which the lists are in
    total, token = total.reshape(G, K * n), token.reshape(G, K * n)
    best, at = total.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :N], at[:, :N]
    short = N - best.shape[1]
    parent, token = at // n, token.gather(1, at)
    best, parent, token = (torch.nn.functional.pad(t, (0, short)) for t in (best, parent, token)) if short else (
        best, parent, token)
    if short:
        best[:, -short:] = -math.inf
    none = best == -math.inf
    return best.float(), parent.masked_fill(none, -1), token.masked_fill(none, -1)


# ----------------------------------------------------------------------------- what it takes


def work(case):
    if case["op"] == "beam":
        size, rows = (2 if case["dtype"] == "bfloat16" else 4), case["groups"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * size + 4) + case["groups"] * case["count"] * 20,
                "flops": 4 * rows * case["vocab"]}
    D, KVH, H, P = HEAD_DIM, case["kv_heads"], case["heads"], case["page"]
    new, past = _lengths(case)
    T = sum(new)
    index = 4 * (2 * len(new) + 1 + sum(-(-(a + b) // P) for a, b in zip(new, past)))
    row = 2 * KVH * (D + 1)  # codes and exponents of a position's keys and values
    if case["op"] == "write":
        table = 2 * 4 * D * T if case["rotate"] else 0
        flops = 3 * T * (H + KVH) * D if case["rotate"] else 0
        return {"bytes": 2 * 2 * T * (H + KVH) * D + 2 * T * KVH * D + T * row + min(table, 2 * 4 * D * 32768) + index
                + 2 * 2 * T * KVH * D, "flops": flops + 4 * T * KVH * D}
    keys = sum(a + b for a, b in zip(new, past))
    if case["op"] == "read":
        return {"bytes": keys * (row + 2 * 2 * KVH * D) + index, "flops": 2 * keys * KVH * D}
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, past))  # (token, key it sees)
    shared = sum(b // P * P for i, b in enumerate(past) if i % case["share"])  # read for the search's first beam
    return {"bytes": (keys - shared) * row + 2 * 2 * T * H * D + index, "flops": 4 * pairs * H * D}


# ----------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    """What run() returns, sequence by sequence and head by head (group by group) from the definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "beam":
        return _exact_beam(case, s)
    new, past = _lengths(case)
    P, H, KVH, D = case["page"], case["heads"], case["kv_heads"], HEAD_DIM

    def held(b, length, kind):
        """Keys or values of a sequence, [KVH, length, D]."""
        at = s["page_table"][b, :-(-length // P)].long()
        codes, e = s[kind + "_pages"][at].double(), s[kind + "_scale"][at].double()
        x = torch.ldexp(codes, (e - 127.0)[..., None])
        return x.transpose(0, 1).reshape(KVH, -1, D)[:, :length]

    if case["op"] == "read":
        both = [[held(b, a + c, kind).transpose(0, 1) for b, (a, c) in enumerate(zip(new, past))] for kind in "kv"]
        return torch.cat(both[0]), torch.cat(both[1])
    if case["op"] == "write":
        x = s["qkv"].double().view(-1, H + 2 * KVH, D)
        if case["rotate"]:
            at = torch.tensor([b + i for a, b in zip(new, past) for i in range(a)], device="cuda")
            z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous())
            turn = torch.complex(s["cos"][at, :D // 2].double(), s["sin"][at, :D // 2].double())
            z[:, :H + KVH] *= turn[:, None]
            x = torch.cat([z.real, z.imag], -1)
        x = x.to(torch.bfloat16).double()
        return x[:, :H], _exact_codes(x[:, H:H + KVH], case["code"]), _exact_codes(x[:, H + KVH:], case["code"])
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    t = 0
    for b, (n, before) in enumerate(zip(new, past)):
        hidden = torch.ones((n, n + before), dtype=torch.bool, device="cuda").triu(before + 1)
        keys, values = held(b, n + before, "k"), held(b, n + before, "v")
        for h in range(H):
            k, v = keys[h // (H // KVH)], values[h // (H // KVH)]
            score = (s["q"][t:t + n, h].double() @ k.T * s["scale"]).masked_fill_(hidden, -math.inf)
            out[t:t + n, h * D:(h + 1) * D] = torch.softmax(score, -1) @ v
        t += n
    return out


def _exact_codes(x, code):
    """The numbers that the codes of x [..., D] stand for."""
    most, digits = (127.0, None) if code == "int8" else (448.0, 3)
    e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True).clamp(min=1e-20) / most))
    y = torch.ldexp(x, -e)
    # the spacing of the codes: 1, or 2^-3 of a number's own power of two, from 2^-6 on downwards the same
    step = 1.0 if digits is None else torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - digits)
    return torch.ldexp(torch.round(y / step) * step, e)  # to even where it lies in the middle


def _exact_beam(case, s):
    G, K, V, N = case["groups"], case["beams"], case["vocab"], case["count"]
    values = torch.full((G, N), -math.inf, dtype=torch.float64, device="cuda")
    parents = torch.full((G, N), -1, dtype=torch.int64, device="cuda")
    tokens = parents.clone()
    for g in range(G):
        total = s["scores"][g].double()[:, None] + torch.log_softmax(s["logits"][g * K:(g + 1) * K].double(), 1)
        total = total.reshape(-1)
        best, at = total.sort(descending=True, stable=True)
        n = min(N, int(total.isfinite().sum()))
        values[g, :n], parents[g, :n], tokens[g, :n] = best[:n], at[:n] // V, at[:n] % V
    return values, parents, tokens
