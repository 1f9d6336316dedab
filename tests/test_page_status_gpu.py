"""The flags of the paged operators are taken whole: none is lost between its reading and its clearing."""

import threading

import pytest
import torch

from test_paged_gpu import Batch
from xb200 import ops

pytestmark = pytest.mark.gpu


def test_no_report_is_lost_to_another_reader():
    """A thread reads the status all the time; of every bad call one of the two readers is told."""
    b = Batch([1, 1], [20, 30], 14, 2, 16, seed=60)
    b.table_dev[0, 0] = b.kp.shape[0]  # outside the pool
    q = b.q.cuda()
    b.attend(q)
    torch.cuda.synchronize()
    ops.page_status()
    told, calls, stop = [0], [0], [False]

    def read():
        with torch.cuda.stream(torch.cuda.Stream()):
            while not stop[0]:
                told[0] += ops.page_status()
                calls[0] += 1

    reader = threading.Thread(target=read)
    reader.start()
    lost = 0
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(400):
                before = told[0]
                b.attend(q)
                torch.cuda.current_stream().synchronize()
                if ops.page_status():
                    continue
                n = calls[0]
                while calls[0] < n + 2:  # the reader has counted what it took meanwhile
                    pass
                lost += told[0] == before
    finally:
        stop[0] = True
        reader.join()
    assert lost == 0
    assert ops.page_status() == 0 and ops.device_status() == 0
