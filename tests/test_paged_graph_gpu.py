"""PagedDecodeGraph: what it prepares before its capture, and what it keeps."""

import gc
import subprocess
import sys
import weakref

import pytest
import torch

from conftest import PKG_ROOT
from xb200.paged import PagedDecodeGraph, PagedKVCache
from xb200.qwen import Qwen2Model, QwenConfig, random_weights

pytestmark = pytest.mark.gpu

CFG = dict(n_layer=1, vocab_size=512)


def _model(rope_len=1024):
    cfg = QwenConfig(**CFG)
    return Qwen2Model(random_weights(cfg, seed=41), cfg, rope_len=rope_len)


def test_the_step_before_the_capture_has_the_captured_sizes():
    """The attention picks its kernel by the table's width: the eager step has to set up the one that is captured."""
    model = _model()
    cache = PagedKVCache(model.cfg, 40, 16)
    seen = []
    forward = model.forward_packed

    def record(ids, c, batch, **kw):
        seen.append((torch.cuda.is_current_stream_capturing(), tuple(ids.shape), tuple(batch.page_table.shape),
                     tuple(batch.kv_len.shape)))
        return forward(ids, c, batch, **kw)

    model.forward_packed = record
    PagedDecodeGraph(model, cache, 3, 200)
    assert [s[0] for s in seen] == [False, True] and seen[0][1:] == seen[1][1:]


WIDE = """
import sys
sys.path.insert(0, {pkg!r})
import torch
from xb200 import ops
from xb200.paged import PagedDecodeGraph, PagedKVCache
from xb200.qwen import Qwen2Model, QwenConfig, random_weights

cfg = QwenConfig(**{cfg!r})
model = Qwen2Model(random_weights(cfg, seed=41), cfg, rope_len=32768)
B = 160
cache, eager = (PagedKVCache(cfg, 4 * B, 16) for _ in range(2))
graph = PagedDecodeGraph(model, cache, B, 32768)  # the first call of the process
one, two = ([c.add() for _ in range(B)] for c in (cache, eager))
toks = torch.arange(B, device="cuda")
for _ in range(3):
    got = graph.step(one, toks)
    want = torch.empty_like(got)
    model.forward_paged(toks, eager, two, next_token=want)
    assert torch.equal(got, want)
    toks = want.clone()
assert ops.device_status() == 0 and ops.page_status() == 0
"""


def test_a_graph_whose_table_takes_64_bit_walks_is_the_first_call_of_a_process():
    """160 sequences of up to 32768 positions: a kernel that smaller steps do not use."""
    got = subprocess.run([sys.executable, "-c", WIDE.format(pkg=PKG_ROOT, cfg=CFG)], capture_output=True, text=True,
                         timeout=300)
    assert got.returncode == 0, got.stderr[-2000:]


def test_a_graph_keeps_its_model():
    """The captured kernels read the model's weights and tables: they live as long as the graph."""
    model = _model()
    cache, eager = (PagedKVCache(model.cfg, 8, 16) for _ in range(2))
    graph = PagedDecodeGraph(model, cache, 2, 64)
    toks = torch.tensor([3, 4], device="cuda")
    want = torch.empty_like(toks)
    model.forward_paged(toks, eager, [eager.add(), eager.add()], next_token=want)
    alive = weakref.ref(model)
    del model
    gc.collect()
    assert alive() is not None
    assert torch.equal(graph.step([cache.add(), cache.add()], toks), want)
