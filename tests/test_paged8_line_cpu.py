"""The split of the work of an attention call over 8-bit pages, run on the host
(tests/paged_line8.cpp): every unit is handed out once, in order, its key tiles
without a gap."""

import ctypes
import os
import random
import subprocess

import numpy as np
import pytest
from test_paged_line_cpu import LAYOUTS, SMS, _batch

from conftest import PKG_ROOT, ROOT


@pytest.fixture(scope="module")
def line(tmp_path_factory):
    so = tmp_path_factory.mktemp("line8") / "line8.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-fwrapv", "-shared", "-fPIC", "-I" + os.path.join(PKG_ROOT, "csrc"),
                    os.path.join(ROOT, "tests", "paged_line8.cpp"), "-o", str(so)], check=True)
    fn = ctypes.CDLL(str(so)).paged_line8
    fn.argtypes = [ctypes.c_int] * 9 + [ctypes.c_void_p] * 2 + [ctypes.c_char_p, ctypes.c_size_t] + [ctypes.c_void_p] * 4

    def run(rows, new, kv_len, H, KVH, page, max_pages, bits=0, q_start=None, T=None):
        starts = np.concatenate([[0], np.cumsum(new)]) if q_start is None else np.array(q_start)
        starts, lens = starts.astype(np.int32), np.array(kv_len, dtype=np.int64).astype(np.int32)
        msg = ctypes.create_string_buffer(400)
        units, weight, bound, wide = ctypes.c_int64(), ctypes.c_double(), ctypes.c_double(), ctypes.c_int()
        rc = fn(rows, int(starts[-1]) if T is None else T, len(lens), KVH, H // KVH, page, max_pages, SMS, bits,
                starts.ctypes.data, lens.ctypes.data, msg, 400, ctypes.addressof(units), ctypes.addressof(weight),
                ctypes.addressof(bound), ctypes.addressof(wide))
        assert (rc == 0) == (msg.value == b"")
        return msg.value.decode(), units.value, weight.value, bound.value, bool(wide.value)

    return run


@pytest.mark.parametrize("short", [False, True])
@pytest.mark.parametrize("seed", range(60))
def test_every_unit_once(line, seed, short):
    rnd = random.Random(2000 + seed)
    H, KVH = LAYOUTS[seed % len(LAYOUTS)]
    new, lens = _batch(rnd, short)
    page = rnd.choice([8, 16, 48])
    cols = -(-max(lens + [1]) // page) + rnd.randrange(3)
    rep = H // KVH
    for rows in (8, 16):
        if rep > rows:
            continue
        tpt = rows // rep
        want = KVH * sum(32 + max(0, n_kv - n + min(n, t + tpt)) for n, n_kv in zip(new, lens) for t in range(0, n, tpt))
        for bits in (0, 32, 64):
            wrong, units, weight, bound, _ = line(rows, new, lens, H, KVH, page, cols, bits)
            assert wrong == "" and weight == want and weight <= bound
            assert units == KVH * sum(-(-n // tpt) for n in new)


@pytest.mark.parametrize("rows,T,H,KVH,kv_len", [(16, 330_000, 12, 12, 500), (8, 200_000, 8, 8, 1024), (16, 90_000, 16, 1, 0)])
def test_more_new_tokens_than_keys(line, rows, T, H, KVH, kv_len):
    wrong, units, weight, bound, wide = line(rows, [T], [kv_len], H, KVH, 16, max(1, kv_len // 16))
    assert wrong == "" and weight <= bound and units == KVH * -(-T // (rows // (H // KVH)))


@pytest.mark.parametrize("rows", [8, 16])
def test_positions_up_to_the_last_that_is_accepted(line, rows):
    top = 2 ** 31 - 8
    for lens in ([top], [top - 200, 5, top]):
        wrong, units, weight, bound, wide = line(rows, [20] * len(lens), lens, 8, 4, 8, top // 8)
        assert wrong == "" and wide and weight <= bound and units == 4 * len(lens) * -(-20 // (rows // 2))
