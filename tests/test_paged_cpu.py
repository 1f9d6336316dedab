"""Host side of the paged KV cache: argument checks of the C entry points and page bookkeeping (no GPU)."""

import ctypes

import pytest
import torch

from xb200 import _lib, ops
from xb200._lib import XbError


def _i32(*v):
    return (ctypes.c_int32 * len(v))(*v)


def _copy(src, dst, n_pages=8, outer=2, page_bytes=64, outer_bytes=None, base=1 << 20):
    s, d = _i32(*src), _i32(*dst)
    _lib.call("xb_copy_pages", base, outer, n_pages * page_bytes if outer_bytes is None else outer_bytes, n_pages,
              page_bytes, ctypes.addressof(s), ctypes.addressof(d), len(src), None)


@pytest.mark.parametrize("src,dst,code,text", [
    ([0], [8], _lib.XB_ERR_INVALID, "destination outside"),
    ([8], [0], _lib.XB_ERR_INVALID, "source outside"),
    ([0], [-1], _lib.XB_ERR_INVALID, "destination outside"),
    ([-2 ** 31], [1], _lib.XB_ERR_INVALID, "source outside"),
    ([0, 1], [3, 3], _lib.XB_ERR_INVALID, "twice"),
    ([0, 3], [3, 4], _lib.XB_ERR_INVALID, "both"),
    ([5], [5], _lib.XB_ERR_INVALID, "both"),
    ([0] * 9, list(range(1, 8)) + [1, 2], _lib.XB_ERR_INVALID, "pool of 8"),
])
def test_copy_pages_refuses_bad_lists(src, dst, code, text):
    with pytest.raises(XbError) as e:
        _copy(src, dst)
    assert e.value.code == code and text in e.value.message


@pytest.mark.parametrize("kw", [dict(page_bytes=24), dict(outer_bytes=100), dict(base=8), dict(outer_bytes=256),
                                dict(outer=70000)])
def test_copy_pages_refuses_layouts(kw):
    with pytest.raises(XbError) as e:
        _copy([0], [1], **kw)
    assert e.value.code == _lib.XB_ERR_UNSUPPORTED


def test_copy_pages_without_work_is_a_no_op():
    _lib.call("xb_copy_pages", None, 4, 64, 8, 64, None, None, 0, None)
    _copy([0], [1], outer=0)


_KV = dict(k=1 << 13, v=1 << 14, table=1 << 16, q_start=1 << 17, kv_len=1 << 18, n_pages=10, n_kv_head=2, page_size=16,
           head_dim=64, batch=2, max_pages=3, ld_table=3, k_page=2048, k_head=1024, k_row=64, v_page=2048, v_head=1024,
           v_row=64)


def _split(args, kw):
    """The call's arguments and its packed xb_paged_kv, with `kw` over the defaults of either."""
    kv = {k: kw.get(k, v) or 0 for k, v in _KV.items()}
    assert set(kw) <= set(args) | set(_KV)
    return {k: kw.get(k, v) for k, v in args.items()}, ops._PAGED_KV(*kv.values())


def _attn(**kw):
    a, kv = _split(dict(q=1 << 12, out=1 << 15, tokens=4, n_head=14, ld_q=896, ld_out=896, scale=0.125, ws=None,
                        ws_bytes=0), kw)
    _lib.call("xb_paged_attention_bf16", a["q"], a["out"], kv, *list(a.values())[2:], None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(n_head=13), _lib.XB_ERR_INVALID, "shape"),
    (dict(tokens=-1), _lib.XB_ERR_INVALID, "shape"),
    (dict(batch=-1), _lib.XB_ERR_INVALID, "shape"),
    (dict(max_pages=0), _lib.XB_ERR_INVALID, "shape"),
    (dict(ld_table=2), _lib.XB_ERR_INVALID, "shape"),
    (dict(n_pages=0), _lib.XB_ERR_INVALID, "shape"),
    (dict(page_size=12), _lib.XB_ERR_UNSUPPORTED, "multiple of 8"),
    (dict(head_dim=128), _lib.XB_ERR_UNSUPPORTED, "head_dim"),
    (dict(k_row=60), _lib.XB_ERR_UNSUPPORTED, "strides"),
    (dict(v_page=0), _lib.XB_ERR_UNSUPPORTED, "strides"),
    (dict(max_pages=1 << 28, ld_table=1 << 28), _lib.XB_ERR_UNSUPPORTED, "positions"),
    (dict(scale=0.0), _lib.XB_ERR_INVALID, "scale"),
    (dict(scale=-1.0), _lib.XB_ERR_INVALID, "scale"),
    (dict(scale=float("nan")), _lib.XB_ERR_INVALID, "scale"),
    (dict(scale=float("inf")), _lib.XB_ERR_INVALID, "scale"),
    (dict(n_head=258), _lib.XB_ERR_UNSUPPORTED, "heads per KV head"),
    (dict(q=None), _lib.XB_ERR_INVALID, "null"),
    (dict(table=None), _lib.XB_ERR_INVALID, "null"),
    (dict(ld_q=895), _lib.XB_ERR_INVALID, "pitch"),
    (dict(ld_out=900), _lib.XB_ERR_UNSUPPORTED, "16-byte"),
    (dict(q=4100), _lib.XB_ERR_UNSUPPORTED, "16-byte"),
    (dict(), _lib.XB_ERR_INVALID, "workspace"),
])
def test_paged_attention_refuses(kw, code, text):
    with pytest.raises(XbError) as e:
        _attn(**kw)
    assert e.value.code == code and text in e.value.message, e.value.message


def test_paged_attention_without_work_is_a_no_op():
    _attn(tokens=0, q=None, out=None)
    _attn(batch=0, kv_len=None)


def _rope(**kw):
    a, kv = _split(dict(qkv=1 << 12, cos=1 << 11, sin=1 << 10, q=1 << 15, tokens=4, n_head=14, rope_rows=64,
                        ld_qkv=18 * 64, ld_q=896), kw)
    v = list(a.values())
    _lib.call("xb_paged_rope_kv_bf16", *v[:4], kv, *v[4:], None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(head_dim=80), _lib.XB_ERR_UNSUPPORTED, "head_dim"),
    (dict(head_dim=96), _lib.XB_ERR_UNSUPPORTED, "head_dim"),
    (dict(head_dim=1024), _lib.XB_ERR_UNSUPPORTED, "head_dim"),
    (dict(cos=None), _lib.XB_ERR_INVALID, "null"),
    (dict(ld_qkv=17 * 64), _lib.XB_ERR_INVALID, "pitch"),
    (dict(ld_q=900), _lib.XB_ERR_UNSUPPORTED, "16-byte"),
    (dict(n_kv_head=0), _lib.XB_ERR_INVALID, "shape"),
    (dict(page_size=20), _lib.XB_ERR_UNSUPPORTED, "multiple of 8"),
])
def test_paged_rope_kv_refuses(kw, code, text):
    with pytest.raises(XbError) as e:
        _rope(**kw)
    assert e.value.code == code and text in e.value.message, e.value.message


def test_operators_refuse_host_tensors():
    x = torch.zeros((1, 2, 8, 2, 16, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.copy_pages(x, [0], [1])
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(x[0, 0, :, 0], x[0, 0], x[0, 1], x[0, 0, :, 0], i.view(1, 2), i, i[:1], 1.0)


# ----------------------------------------------------------------------------- page bookkeeping


class _Cfg:
    n_layer, n_kv_head, head_dim = 2, 2, 16


@pytest.fixture
def copies(monkeypatch):
    """ops.copy_pages on host tensors; the calls are recorded."""
    calls = []

    def copy(pages, src, dst, dim=2):
        src, dst = list(src), list(dst)
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        pages[:, :, dst] = pages[:, :, src]
        calls.append((src, dst))
        return pages

    monkeypatch.setattr(ops, "copy_pages", copy)
    return calls


def _cache(n=12, page=8):
    from xb200.paged import PagedKVCache

    return PagedKVCache(_Cfg, n, page, device="cpu")


def _check(cache):
    """Reference counts are the sequences' uses, and the free pages are the unused ones."""
    uses = [0] * cache.n_pages
    for s in cache._seqs.values():
        assert len(s.pages) == -(-s.length // cache.page_size)
        for p in s.pages:
            uses[p] += 1
    assert uses == cache._refs
    assert sorted(cache._free) == [p for p, n in enumerate(uses) if n == 0]


def _write(cache, batch, seqs, counts, value):
    """What a step's RoPE operator does: the position's value in every new position's page."""
    start = batch.q_start.tolist()
    for i, _ in enumerate(seqs):
        for t in range(start[i], start[i + 1]):
            p = int(batch.positions[t])
            assert p == int(batch.kv_len[i]) - (start[i + 1] - t)
            cache.pages[:, :, int(batch.page_table[i, p // cache.page_size]), :, p % cache.page_size] = value(i, p)


def _read(cache, seq):
    """The first element of every position of layer 0's keys."""
    P = cache.page_size
    return [float(cache.pages[0, 0, cache.page_ids(seq)[p // P], 0, p % P, 0]) for p in range(cache.length(seq))]


def test_steps_tables_and_positions(copies):
    c = _cache()
    a, b = c.add(), c.add()
    s = c.step([a, b], [10, 3])
    assert s.page_table.tolist() == [[0, 1], [2, 0]] and s.kv_len.tolist() == [10, 3]
    assert s.q_start.tolist() == [0, 10, 13] and s.last.tolist() == [9, 12]
    assert s.positions.tolist() == list(range(10)) + [0, 1, 2]
    s = c.step([b, a])
    assert s.last is None and s.q_start.tolist() == [0, 1, 2] and s.positions.tolist() == [3, 10]
    assert s.page_table.dtype == torch.int32 and s.positions.dtype == torch.int64
    _check(c)
    assert not copies


def test_fork_copies_the_page_that_both_write(copies):
    c = _cache()
    a = c.add()
    _write(c, c.step([a], [11]), [a], [11], lambda i, p: p)
    b = c.fork(a)
    d = c.fork(a)
    assert c.free_pages == 10 and not copies
    _write(c, c.step([a, b, d]), [a, b, d], [1] * 3, lambda i, p: 30 * (i + 1) + p)
    assert copies == [([1, 1], [2, 3])]  # the last sharer writes in place
    assert _read(c, a) == list(range(11)) + [41] and _read(c, b) == list(range(11)) + [71]
    assert _read(c, d) == list(range(11)) + [101]
    assert c.page_ids(a)[0] == c.page_ids(b)[0] == c.page_ids(d)[0]
    _check(c)
    c.free(a)
    _check(c)
    assert _read(c, b) == list(range(11)) + [71]


def test_fork_at_a_page_end_copies_nothing(copies):
    c = _cache()
    a = c.add()
    c.step([a], [8])
    b = c.fork(a)
    c.step([a, b])
    assert not copies and c.page_ids(a)[1] != c.page_ids(b)[1]
    empty = c.fork(c.add())
    assert c.length(empty) == 0
    _check(c)


def test_a_step_that_does_not_fit_changes_nothing(copies):
    c = _cache(n=4)
    a = c.add()
    c.step([a], [12])
    b = c.fork(a)
    before = (c.page_ids(a), c.page_ids(b), c.free_pages)
    with pytest.raises(RuntimeError, match="full"):
        c.step([a, b], [21, 2])  # a copy and three fresh pages
    assert before == (c.page_ids(a), c.page_ids(b), c.free_pages) and c.length(a) == 12 and not copies
    c.step([a, b], [1, 1])
    _check(c)


def test_truncate_gives_pages_back(copies):
    c = _cache()
    a = c.add()
    c.step([a], [30])
    b = c.fork(a)
    c.truncate(a, 9)
    assert c.length(a) == 9 and len(c.page_ids(a)) == 2 and c.length(b) == 30
    _check(c)
    c.truncate(b, 0)
    assert c.page_ids(b) == []
    with pytest.raises(ValueError):
        c.truncate(a, 10)
    _check(c)


def test_compact_moves_high_pages_down(copies):
    c = _cache(n=20)
    seqs = [c.add() for _ in range(5)]
    _write(c, c.step(seqs, [20, 9, 8, 25, 4]), seqs, None, lambda i, p: 50 * i + p)
    fork = c.fork(seqs[3])
    c.free(seqs[0])
    c.free(seqs[2])
    moved = c.compact()
    assert moved > 0 and sorted(p for s in c._seqs.values() for p in set(s.pages))[-1] == 20 - c.free_pages - 1
    assert _read(c, seqs[1]) == [50 + p for p in range(9)] and _read(c, seqs[4]) == [200 + p for p in range(4)]
    assert _read(c, fork) == _read(c, seqs[3]) == [150 + p for p in range(25)]
    _check(c)
    assert c.compact() == 0
    c.step([fork, seqs[3]])
    _check(c)


def test_random_histories_keep_the_books(copies):
    import random

    for seed in range(30):
        rnd = random.Random(seed)
        c = _cache(n=rnd.randint(3, 25))
        want = {}
        tick = 0
        for _ in range(60):
            op = rnd.choice(["add", "fork", "free", "step", "step", "step", "truncate", "compact"])
            live = list(want)
            if op == "add":
                want[c.add()] = []
            elif op == "compact":
                c.compact()
            elif live:
                q = rnd.choice(live)
                if op == "fork":
                    want[c.fork(q)] = list(want[q])
                elif op == "free":
                    c.free(q)
                    del want[q]
                elif op == "truncate":
                    n = rnd.randint(0, len(want[q]))
                    c.truncate(q, n)
                    del want[q][n:]
                else:
                    seqs = rnd.sample(live, rnd.randint(1, len(live)))
                    counts = [rnd.randint(1, 12) for _ in seqs]
                    try:
                        b = c.step(seqs, counts)
                    except RuntimeError:
                        b = None
                    if b is not None:
                        tick = (tick + 1) % 100  # exact in bf16 with the sequence's place
                        _write(c, b, seqs, counts, lambda i, p: tick + i / 64)
                        for i, (s, n) in enumerate(zip(seqs, counts)):
                            want[s] += [float(torch.tensor(tick + i / 64).to(torch.bfloat16))] * n
            _check(c)
            for s, w in want.items():
                assert _read(c, s) == w


def test_cache_refusals(copies):
    from xb200.paged import PagedKVCache

    c = _cache()
    a = c.add()
    for bad in ([], [a, a]):
        with pytest.raises(ValueError):
            c.step(bad)
    with pytest.raises(ValueError):
        c.step([a], [0])
    with pytest.raises(ValueError):
        c.step([a], [1, 1])
    with pytest.raises(KeyError):
        c.step([a, 99])
    c.free(a)
    with pytest.raises(KeyError):
        c.free(a)
    with pytest.raises(KeyError):
        c.length(a)
    for n, p in ((0, 8), (4, 12), (4, 0)):
        with pytest.raises(ValueError):
            PagedKVCache(_Cfg, n, p, device="cpu")


def test_fresh_slots_and_taken_workspaces():
    a, b = ops.fresh_slot(), ops.fresh_slot()
    assert a != b
    with ops.workspace_slot(a):
        key = (torch.device("cuda:0"), a)
        ops._workspaces[key] = "buffer"
        assert ops.take_workspace("cuda:0") == "buffer" and key not in ops._workspaces
        assert ops.take_workspace("cuda:0") is None


def test_more_sequences_than_a_kernel_scans_are_refused():
    """Every CTA scans all sequences with 32-bit counters, and a run of empty ones is passed while others wait."""
    for call in (_attn, _rope):
        for batch in ((1 << 20) + 1, 2 ** 31 - 2):
            with pytest.raises(XbError) as e:
                call(batch=batch)
            assert e.value.code == _lib.XB_ERR_UNSUPPORTED and "2^20 sequences" in e.value.message, e.value.message


def test_a_copy_that_fails_leaves_the_books(copies, monkeypatch):
    c = _cache()
    a = c.add()
    _write(c, c.step([a], [11]), [a], [11], lambda i, p: p)
    b = c.fork(a)
    before = (c.page_ids(a), c.page_ids(b), list(c._refs), sorted(c._free))

    def fails(*args, **kw):
        raise RuntimeError("no copy")

    with monkeypatch.context() as m:
        m.setattr(ops, "copy_pages", fails)
        with pytest.raises(RuntimeError, match="no copy"):
            c.step([b, a], [9, 3])
    assert before == (c.page_ids(a), c.page_ids(b), c._refs, sorted(c._free)) and c.length(a) == c.length(b) == 11
    _check(c)
    _write(c, c.step([b, a], [9, 3]), [b, a], [9, 3], lambda i, p: 50 * (i + 1) + p)
    assert _read(c, b) == list(range(11)) + [50 + p for p in range(11, 20)]
    assert _read(c, a) == list(range(11)) + [100 + p for p in range(11, 14)]
    _check(c)


def test_copy_pages_refuses_pages_of_2_36_bytes():
    with pytest.raises(XbError) as e:
        _copy([0], [1], n_pages=2, page_bytes=1 << 36)
    assert e.value.code == _lib.XB_ERR_UNSUPPORTED


def test_a_scale_whose_base_2_form_overflows_is_refused():
    """scores are scaled by scale * log2(e) in fp32: infinite from 2.4e38 on, and then every score of zero is NaN."""
    for scale, refused in ((2.35e38, False), (2.37e38, True), (3e38, True)):
        with pytest.raises(XbError) as e:  # without a workspace: nothing is launched
            _attn(scale=scale)
        assert ("scale" in e.value.message) == refused, e.value.message


@pytest.mark.parametrize("page_size", [0, -16, 12])
def test_generation_refuses_a_page_size_as_the_cache_does(page_size):
    from xb200.paged import generate_paged

    class Model:
        cfg, position_limit, device = _Cfg, 64, torch.device("cpu")

    with pytest.raises(ValueError, match="multiple of 8"):
        generate_paged(Model, [torch.ones(3, dtype=torch.int64)], 4, page_size=page_size)
