"""The calls that skip the interpreter (csrc/calls.cpp) against the ones that do not: the same results, and
what they do not take goes the other way."""

import pytest
import torch
from test_paged8_gpu import DTYPES, Coded
from test_paged_gpu import Batch

from xb200 import ops

pytestmark = pytest.mark.gpu


class _Aside:
    """Every call is left alone."""

    paged_attention = paged_rope_kv = paged_read_kv = staticmethod(lambda *a: False)
    beam_select = staticmethod(lambda *a: None)


def _both(monkeypatch, run):
    """Results and pools of the direct way, then of the other one."""
    out = [run()]
    with monkeypatch.context() as m:
        m.setattr(ops, "_calls", _Aside)
        out.append(run())
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, *DTYPES])
@pytest.mark.parametrize("new,H,KVH,layout", [([1], 14, 2, "nhpd"), ([1, 3, 0, 1], 14, 2, "joint"), ([70, 2], 12, 12, "rows"),
                                              ([1], 1, 1, "nhpd")])
def test_the_same_with_and_without(new, H, KVH, layout, dtype, monkeypatch):
    coded = dtype is not torch.bfloat16

    def run():
        a = (new, [5 * i for i in range(len(new))], H, KVH, 16)
        b = Coded(dtype, *a, seed=80, layout=layout) if coded else Batch(*a, seed=80, layout=layout)
        ex = (b.ks, b.vs) if coded else ()
        at = (b.table_dev, b.q_start, b.kv_len)
        T = sum(new)
        qkv = torch.randn((T, (H + 2 * KVH) * 64), generator=torch.Generator().manual_seed(81)).to(torch.bfloat16).cuda()
        cos, sin = (torch.randn((40 + max(new), 64), generator=torch.Generator().manual_seed(82)).cuda() for _ in range(2))
        q, out = (torch.zeros((T, H, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        k, v = (torch.zeros((T, KVH, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        assert ops.paged_rope_kv(qkv, cos, sin, q, b.kp, b.vp, *at, *ex) is q
        assert ops.paged_attention(q, b.kp, b.vp, out, *at, 0.125, *ex) is out
        assert ops.paged_read_kv(k, v, b.kp, b.vp, *at, *ex) == (k, v)
        direct = ops._calls
        if direct is not _Aside:  # these are calls that it takes
            assert direct.paged_rope_kv(qkv, cos, sin, q, b.kp, b.vp, *at, *(ex or (None, None))) is True
            assert direct.paged_attention(q, b.kp, b.vp, out, *at, 0.125, *(ex or (None, None))) is True
            assert direct.paged_read_kv(k, v, b.kp, b.vp, *at, *(ex or (None, None))) is True
        return [x.view(torch.uint8) for x in (q, out, k, v, b.kp, b.vp, *ex)]

    ops._direct()
    here, there = _both(monkeypatch, run)
    assert all(torch.equal(x, y) for x, y in zip(here, there)) and ops.page_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_selection_with_and_without(dtype, monkeypatch):
    x = torch.randn((12, 5000), generator=torch.Generator().manual_seed(83)).to(dtype).cuda()
    scores = torch.randn((3, 4), generator=torch.Generator().manual_seed(84)).cuda()
    ops._direct()
    assert ops._calls.beam_select(x, scores, 8) is not None
    here, there = _both(monkeypatch, lambda: ops.beam_select(x, scores, 8))
    for a, b in zip(here, there):
        assert torch.equal(a, b) and a.dtype is b.dtype and a.shape == b.shape == (3, 8)


def test_what_is_left_alone():
    """Other types, shapes, strides and devices, and what the library refuses: nothing is launched."""
    b = Coded(torch.int8, [1, 2], [40, 25], 14, 2, 16, seed=85)
    direct = ops._direct()
    q, out = b.q.cuda(), torch.full((3, 14 * 64), 7.0, dtype=torch.bfloat16, device="cuda")
    good = [q, b.kp, b.vp, out, b.table_dev, b.q_start, b.kv_len, 0.125, b.ks, b.vs]
    bf16 = torch.zeros_like(b.kp, dtype=torch.bfloat16)
    other = [(0, q.cpu()), (0, q.float()), (0, q[:2]), (0, q.flatten(1)), (0, None), (0, 3), (1, b.kp[:, :1]),
             (1, b.kp.view(torch.float8_e4m3fn)), (1, b.kp.transpose(0, 1)), (1, bf16), (3, q), (3, out[:, :64]),
             (3, out.float()), (4, b.table_dev.long()), (4, b.table_dev[:1]), (4, b.table_dev.t().contiguous().t()),
             (5, b.q_start[:2]), (6, b.kv_len.cpu()), (7, "x"), (7, 1), (7, -1.0), (7, float("nan")), (8, None), (9, None),
             (8, b.ks.view(torch.int8)), (8, b.ks[:, :, :8]), (9, b.vs.transpose(1, 2).contiguous().transpose(1, 2))]
    for i, x in other:
        args = list(good)
        args[i] = x
        assert direct.paged_attention(*args) is False, (i, x)
    assert direct.paged_attention(*good[:9]) is False
    assert bool((out == 7).all())
    logits, scores = torch.randn((6, 100), device="cuda"), torch.zeros((2, 3), device="cuda")
    for args in ((logits.half(), scores, 4), (logits, scores.double(), 4), (logits, scores[:1], 4), (logits, scores, 0),
                 (logits, scores, 65), (logits, scores, 1 << 70), (logits, scores, 4.0), (logits.cpu(), scores, 4),
                 (logits.t().contiguous().t(), scores, 4), (logits, scores.view(-1), 4), (None, scores, 4), (logits, scores)):
        assert direct.beam_select(*args) is None
    assert ops.device_status() == 0 and ops.page_status() == 0

