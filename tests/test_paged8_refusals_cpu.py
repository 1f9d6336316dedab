"""What the attention over 8-bit pages refuses, it refuses before its first launch (no GPU:
a launch would be answered with an error of CUDA's)."""

import pytest
from test_paged8_cpu import _attn

from xb200 import _lib


@pytest.mark.parametrize("dtype", [2, 5])
@pytest.mark.parametrize("kw,text", [
    (dict(tokens=1 << 20, n_head=128, n_kv_head=1, batch=1 << 20, max_pages=1 << 27, ld_table=1 << 27, page_size=8), "many"),
    # a page of the expanded pool as long as no page may be
    (dict(tokens=64, n_head=65535, n_kv_head=65535, batch=1, max_pages=1, page_size=1 << 17), "strides"),
])
def test_refused_before_the_expansion(kw, text, dtype):
    row = 64 * kw["n_head"]
    with pytest.raises(_lib.XbError) as e:
        _attn(**kw, dtype=dtype, ld_q=row, ld_out=row, ws=1 << 22, ws_bytes=1 << 62, n_pages=1)
    assert e.value.code == _lib.XB_ERR_UNSUPPORTED and text in e.value.message, e.value.message
