"""Errors of CUDA's under the calls that skip the interpreter (csrc/calls.cpp): an entry point
that reports one, after whatever it has launched, is called once and its error raised.  The
entry points are stand-ins that launch nothing."""

import ctypes

import pytest
import torch

from xb200 import _lib, ops

pytestmark = pytest.mark.gpu

P, I, Z = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t
ENTRIES = {  # all but the last two arguments, the text of an error and its length
    "xb_paged_attention_bf16": [P, P, P, I, I, I, I, ctypes.c_float, P, Z, P],
    "xb_paged_attention_q8": [P, P, P, I, I, I, I, ctypes.c_float, P, Z, P],
    "xb_paged_rope_kv_bf16": [P, P, P, P, P, I, I, I, I, I, P],
    "xb_paged_rope_kv_q8": [P, P, P, P, P, I, I, I, I, I, P],
    "xb_paged_read_kv": [P, P, P, I, I, I, P],
    "xb_beam_select": [P, P, I, I, I, I, I, I, ctypes.c_int, P, P, P, P, Z, P],
    "xb_beam_select_workspace_size": [I, I, I, I, P],
    "xb_paged_attention_workspace_size": [I, I, I, I, P],
}


def _call(name):
    bf16 = dict(dtype=torch.bfloat16, device="cuda")
    if name.startswith("xb_beam"):
        return ops.beam_select(torch.zeros((2, 9), device="cuda"), torch.zeros((1, 2), device="cuda"), 2)
    coded = name.endswith("q8")
    kp, vp = (torch.zeros((2, 1, 8, 64), dtype=torch.int8 if coded else torch.bfloat16, device="cuda") for _ in range(2))
    ex = [torch.zeros((2, 1, 8), dtype=torch.uint8, device="cuda") for _ in range(2)] if coded else []
    table, q_start, kv_len = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([[0]], [0, 1], [1]))
    q = torch.zeros((1, 1, 64), **bf16)
    out = torch.full((1, 1, 64), 7.0, **bf16)
    if "attention" in name:
        ops.paged_attention(q, kp, vp, out, table, q_start, kv_len, 0.125, *ex)
    elif "rope" in name:
        ops.paged_rope_kv(torch.zeros((1, 192), **bf16), None, None, out, kp, vp, table, q_start, kv_len, *ex)
    else:
        ops.paged_read_kv(q, out, kp, vp, table, q_start, kv_len)
    return out


@pytest.mark.parametrize("code", [_lib.XB_ERR_CUDA, _lib.XB_ERR_TIMEOUT, -99])
@pytest.mark.parametrize("name", ENTRIES)
def test_an_error_of_cuda_is_raised_and_the_call_not_made_again(name, code, monkeypatch):
    calls = []

    def entry(*a):
        calls.append(name)
        ctypes.memmove(a[-2], b"no such luck\0", 13)
        return code

    fake = ctypes.CFUNCTYPE(ctypes.c_int, *ENTRIES[name], P, Z)(entry)

    class Library:
        def __getattr__(self, what):
            return fake if what == name else getattr(real, what)

    _call(name)  # what the real one needs once is there
    real, before = _lib.load(), ops.launch_count()
    try:
        with monkeypatch.context() as m:
            m.setattr(_lib, "load", Library)
            m.setattr(ops, "_calls", None)
            with pytest.raises(_lib.XbError, match="no such luck") as e:
                _call(name)
            ops._calls = None
    finally:
        ops._calls = None  # bound to the real ones with the next call
    assert e.value.code == code and e.value.func == name and calls == [name]
    assert ops.launch_count() == before
    _call(name)
    assert ops.device_status() == 0
    ops.page_status()
