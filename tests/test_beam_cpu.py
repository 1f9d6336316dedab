"""Argument checks of the beam selection's C entry points (no GPU)."""

import ctypes

import pytest

from xb200 import _lib
from xb200._lib import XbError


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
    sizes = []
    for groups in (1, 4, 40, 4000):
        _lib.call("xb_beam_select_workspace_size", groups, 4, 151936, 8, ctypes.byref(need))
        sizes.append(need.value)
        assert need.value >= groups * 4 * (8 * 8 + 8)
    assert sizes == sorted(sizes)
