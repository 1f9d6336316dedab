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


def _attn(**kw):
    a = dict(q=1 << 12, k=1 << 13, v=1 << 14, out=1 << 15, table=1 << 16, q_start=1 << 17, kv_len=1 << 18, tokens=4,
             batch=2, n_head=14, n_kv_head=2, head_dim=64, n_pages=10, page_size=16, max_pages=3, ld_q=896, ld_out=896,
             ld_table=3, k_page=2048, k_head=1024, k_row=64, v_page=2048, v_head=1024, v_row=64, scale=0.125, ws=None,
             ws_bytes=0)
    a.update(kw)
    _lib.call("xb_paged_attention_bf16", *a.values(), None)


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
    a = dict(qkv=1 << 12, cos=1 << 11, sin=1 << 10, q=1 << 15, k=1 << 13, v=1 << 14, table=1 << 16, q_start=1 << 17,
             kv_len=1 << 18, tokens=4, batch=2, n_head=14, n_kv_head=2, head_dim=64, n_pages=10, page_size=16,
             max_pages=3, rope_rows=64, ld_qkv=18 * 64, ld_q=896, ld_table=3, k_page=2048, k_head=1024, k_row=64,
             v_page=2048, v_head=1024, v_row=64)
    a.update(kw)
    _lib.call("xb_paged_rope_kv_bf16", *a.values(), None)


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
