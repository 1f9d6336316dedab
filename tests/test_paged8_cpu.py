"""Argument checks of the 8-bit paged operators' C entry points (no GPU)."""

import ctypes

import pytest
import torch
from test_paged_cpu import _KV

from xb200 import _lib, ops
from xb200._lib import XbError

_EX = dict(ks=1 << 19, vs=1 << 20, ks_page=32, ks_head=16, vs_page=32, vs_head=16, dtype=2)


def _split(args, kw):
    kv = {k: kw.get(k, v) or 0 for k, v in _KV.items()}
    ex = {k: kw.get(k, v) or 0 for k, v in _EX.items()}
    assert set(kw) <= set(args) | set(_KV) | set(_EX)
    return {k: kw.get(k, v) for k, v in args.items()}, ops._PAGED_KV(*kv.values()) + ops._EXPONENTS(*ex.values())


def _attn(**kw):
    a, kv = _split(dict(q=1 << 12, out=1 << 15, tokens=4, n_head=14, ld_q=896, ld_out=896, scale=0.125, ws=None,
                        ws_bytes=0), kw)
    _lib.call("xb_paged_attention_q8", a["q"], a["out"], kv, *list(a.values())[2:], None)


def _rope(**kw):
    a, kv = _split(dict(qkv=1 << 12, cos=1 << 11, sin=1 << 10, q=1 << 15, tokens=4, n_head=14, rope_rows=64,
                        ld_qkv=18 * 64, ld_q=896), kw)
    v = list(a.values())
    _lib.call("xb_paged_rope_kv_q8", *v[:4], kv, *v[4:], None)


def _read(**kw):
    a, kv = _split(dict(k_out=1 << 12, v_out=1 << 15, tokens=4, ld_k=128, ld_v=128), kw)
    v = list(a.values())
    _lib.call("xb_paged_read_kv", *v[:2], kv, *v[2:], None)


COMMON = [
    (dict(dtype=0), _lib.XB_ERR_UNSUPPORTED, "dtype"),
    (dict(dtype=1), _lib.XB_ERR_UNSUPPORTED, "dtype"),
    (dict(k_row=72), _lib.XB_ERR_UNSUPPORTED, "multiples of 16"),
    (dict(v_head=1032), _lib.XB_ERR_UNSUPPORTED, "multiples of 16"),
    (dict(ks_page=36), _lib.XB_ERR_UNSUPPORTED, "multiples of 8"),
    (dict(vs_head=0), _lib.XB_ERR_UNSUPPORTED, "multiples of 8"),
    (dict(ks=None), _lib.XB_ERR_INVALID, "null"),
    (dict(vs=None), _lib.XB_ERR_INVALID, "null"),
    (dict(vs=(1 << 20) + 4), _lib.XB_ERR_UNSUPPORTED, "8-byte"),
    (dict(table=None), _lib.XB_ERR_INVALID, "null"),
    (dict(tokens=-1), _lib.XB_ERR_INVALID, "shape"),
    (dict(page_size=12), _lib.XB_ERR_UNSUPPORTED, "multiple of 8"),
    (dict(batch=(1 << 20) + 1), _lib.XB_ERR_UNSUPPORTED, "sequences"),
]


@pytest.mark.parametrize("kw,code,text", COMMON + [
    (dict(n_head=13), _lib.XB_ERR_INVALID, "shape"),
    (dict(head_dim=128), _lib.XB_ERR_UNSUPPORTED, "head_dim"),
    (dict(scale=0.0), _lib.XB_ERR_INVALID, "scale"),
    (dict(scale=float("nan")), _lib.XB_ERR_INVALID, "scale"),
    (dict(n_head=258), _lib.XB_ERR_UNSUPPORTED, "heads per KV head"),
    (dict(q=None), _lib.XB_ERR_INVALID, "null"),
    (dict(ld_q=895), _lib.XB_ERR_INVALID, "pitch"),
    (dict(ld_out=900), _lib.XB_ERR_UNSUPPORTED, "16-byte"),
    (dict(), _lib.XB_ERR_INVALID, "workspace"),
    (dict(ws=1 << 22, ws_bytes=1000), _lib.XB_ERR_INVALID, "workspace"),
])
def test_attention_refuses(kw, code, text):
    with pytest.raises(XbError) as e:
        _attn(**kw)
    assert e.value.code == code and text in e.value.message, e.value.message


@pytest.mark.parametrize("kw,code,text", COMMON + [
    (dict(head_dim=80), _lib.XB_ERR_UNSUPPORTED, "head_dim"),
    (dict(cos=None), _lib.XB_ERR_INVALID, "null"),
    (dict(ld_qkv=17 * 64), _lib.XB_ERR_INVALID, "pitch"),
    (dict(ld_q=900), _lib.XB_ERR_UNSUPPORTED, "16-byte"),
])
def test_rope_kv_refuses(kw, code, text):
    with pytest.raises(XbError) as e:
        _rope(**kw)
    assert e.value.code == code and text in e.value.message, e.value.message


@pytest.mark.parametrize("kw,code,text", COMMON[1:] + [
    (dict(head_dim=68), _lib.XB_ERR_UNSUPPORTED, "head_dim"),
    (dict(k_out=None), _lib.XB_ERR_INVALID, "null"),
    (dict(ld_v=120), _lib.XB_ERR_INVALID, "pitch"),
    (dict(ld_k=132), _lib.XB_ERR_UNSUPPORTED, "16-byte"),
    (dict(v_out=4100), _lib.XB_ERR_UNSUPPORTED, "16-byte"),
])
def test_read_kv_refuses(kw, code, text):
    with pytest.raises(XbError) as e:
        _read(**kw)
    assert e.value.code == code and text in e.value.message, e.value.message


def test_null_descriptions_are_refused():
    for name, args in (("xb_paged_attention_q8", (1 << 12, 1 << 15, None, 4, 14, 896, 896, 0.125, None, 0)),
                       ("xb_paged_rope_kv_q8", (1 << 12, None, None, 1 << 15, None, 4, 14, 0, 18 * 64, 896)),
                       ("xb_paged_read_kv", (1 << 12, 1 << 15, None, 4, 128, 128))):
        with pytest.raises(XbError) as e:
            _lib.call(name, *args, None)
        assert e.value.code == _lib.XB_ERR_INVALID and "null" in e.value.message


def test_calls_without_work_are_no_ops():
    _attn(tokens=0, q=None, out=None)
    _attn(batch=0, kv_len=None, ks=None)
    _rope(tokens=0, qkv=None)
    _read(tokens=0, k_out=None, ks=None)
    _read(batch=0, table=None, dtype=0, ks=None, ks_page=0)


def _bytes(*a):
    need = ctypes.c_size_t(0)
    _lib.call("xb_paged_attention_q8_workspace_size", *a, ctypes.byref(need))
    return need.value


def test_workspace_size():
    """As bf16 the pages of a batch of many rows: a slot for each table entry, but no more than the pool has pages."""
    for bad in ((4, 2, 14, 2, 0, 16, 3), (4, 2, 14, 2, 10, 0, 3), (4, 2, 14, 2, 10, 16, 0), (4, 2, 13, 2, 10, 16, 3)):
        with pytest.raises(XbError):
            _bytes(*bad)
    page = 2 * 16 * 64 * 4
    need = ctypes.c_size_t(0)
    _lib.call("xb_paged_attention_workspace_size", 400, 2, 14, 2, ctypes.byref(need))
    small, pool, wide = (_bytes(400, 2, 14, 2, n, 16, c) - need.value for n, c in ((1000, 3), (1000, 600), (1000, 700)))
    assert 6 * page <= small < 7 * page and 1000 * page <= pool <= wide < 1003 * page


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_cache_copies_codes_with_their_exponents(dtype, monkeypatch):
    from test_paged_cpu import _Cfg
    from xb200.paged import PagedKVCache

    calls = []

    def copy(pages, src, dst, dim=2):
        assert pages.is_contiguous() and pages.stride(dim) * pages.element_size() % 16 == 0
        view = pages.view(torch.uint8)
        view.index_copy_(dim, torch.tensor(dst), view.index_select(dim, torch.tensor(src)))
        calls.append((pages.data_ptr(), list(src), list(dst), dim))

    monkeypatch.setattr(ops, "copy_pages", copy)
    c = PagedKVCache(_Cfg, 6, 8, device="cpu", dtype=dtype)
    assert c.pages.dtype is dtype and c.k_scale[1].shape == (6, 2, 8) and c.v_scale[0].dtype is torch.uint8
    a = c.add()
    c.step([a], [11])
    c.pages.view(torch.uint8)[:, :, 1] = 7
    c.k_scale[1][1] = 90
    c.v_scale[0][1] = 91
    b = c.fork(a)
    c.step([b], [1])
    page = c.page_ids(b)[1]
    assert page != 1 and [x[1:] for x in calls] == [([1], [page], 2), ([1], [page], 1)]
    assert bool((c.pages.view(torch.uint8)[:, :, page] == 7).all())
    assert bool((c.k_scale[1][page] == 90).all()) and bool((c.v_scale[0][page] == 91).all())
    c.free(a)
    assert c.compact() == 1 and bool((c.k_scale[1][c.page_ids(b)[1]] == 90).all())
    bf16 = PagedKVCache(_Cfg, 6, 8, device="cpu")
    assert bf16.scales is None and bf16.k_scale == bf16.v_scale == [None, None]
    for bad in (torch.float32, torch.float16, torch.uint8, torch.float8_e5m2):
        with pytest.raises(ValueError, match="bf16, int8"):
            PagedKVCache(_Cfg, 6, 8, device="cpu", dtype=bad)
