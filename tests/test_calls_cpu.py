"""The direct calls (csrc/calls.cpp) where there is no GPU: they take nothing, and the checks one by one answer."""

import pytest
import torch

from xb200 import ops


def test_host_tensors_are_left_alone():
    direct = ops._direct()
    x = torch.zeros((2, 3))
    assert direct.beam_select(x, x, 2) is None
    assert direct.paged_attention(*[x] * 7, 0.5, None, None) is False
    assert direct.paged_rope_kv(x, None, None, *[x] * 6, None, None) is False
    assert direct.paged_read_kv(*[x] * 7, None, None) is False
    assert direct.paged_read_kv() is False and direct.beam_select() is None
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_select(x, x, 2)


def test_bind_wants_every_address():
    direct = ops._direct()
    for bad in ({}, {"xb_beam_select": 1}, 3):
        with pytest.raises((RuntimeError, TypeError)):
            direct.bind(bad)
    ops._calls = None  # bound anew
    assert ops._direct().beam_select(1, 2, 3) is None
