"""The split of a paged attention call's work, run on the host: every unit is
handed out once, in order, its key tiles without a gap, and every part knows
where its unit ends (csrc/paged_walk.cuh, by tests/paged_line.cpp)."""

import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

from conftest import PKG_ROOT, ROOT

SMS = 148


@pytest.fixture(scope="module")
def line(tmp_path_factory):
    so = tmp_path_factory.mktemp("line") / "line.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-fwrapv", "-shared", "-fPIC", "-I" + os.path.join(PKG_ROOT, "csrc"),
                    os.path.join(ROOT, "tests", "paged_line.cpp"), "-o", str(so)], check=True)
    fn = ctypes.CDLL(str(so)).paged_line
    fn.argtypes = [ctypes.c_int] * 9 + [ctypes.c_void_p] * 2 + [ctypes.c_char_p, ctypes.c_size_t] + [ctypes.c_void_p] * 4

    def run(rows, new, kv_len, H, KVH, page, max_pages, bits=0, q_start=None, T=None):
        """(what is wrong or "", units, weight of the line, the host's bound on it, whether the walk has 64 bits)"""
        starts = np.concatenate([[0], np.cumsum(new)]) if q_start is None else np.array(q_start)
        starts, lens = starts.astype(np.int32), np.array(kv_len, dtype=np.int64).astype(np.int32)
        msg = ctypes.create_string_buffer(400)
        units, weight, bound, wide = ctypes.c_int64(), ctypes.c_double(), ctypes.c_double(), ctypes.c_int()
        rc = fn(rows, int(starts[-1]) if T is None else T, len(lens), KVH, H // KVH, page, max_pages,
                SMS if rows <= 16 else 2 * SMS, bits, starts.ctypes.data, lens.ctypes.data, msg, 400,
                ctypes.addressof(units), ctypes.addressof(weight), ctypes.addressof(bound), ctypes.addressof(wide))
        assert (rc == 0) == (msg.value == b"")
        return msg.value.decode(), units.value, weight.value, bound.value, bool(wide.value)

    return run


def _batch(rnd, short):
    """New tokens and lengths of a ragged batch; with `short`, some sequences hold fewer keys than they bring tokens."""
    B = rnd.choice([1, 2, 7, 33, 300])
    most = rnd.choice([1, 5, 40, 700])
    new = [rnd.choice([0, 1, rnd.randint(1, most)]) for _ in range(B)]
    past = rnd.choice([1, 50, 3000, 40000])
    lens = [n + rnd.randrange(past) for n in new]
    if short:
        lens = [rnd.randint(0, n) if rnd.random() < 0.5 else x for n, x in zip(new, lens)]
    return new, lens


LAYOUTS = [(14, 2), (12, 12), (16, 1), (9, 3), (8, 8)]


@pytest.mark.parametrize("seed", range(60))
def test_every_unit_once(line, seed):
    rnd = random.Random(seed)
    H, KVH = LAYOUTS[seed % len(LAYOUTS)]
    new, lens = _batch(rnd, False)
    page = rnd.choice([8, 16, 48])
    cols = -(-max(lens + [1]) // page) + rnd.randrange(3)
    rep = H // KVH
    for rows in (8, 16, 128):
        if rep > rows:
            continue
        got = [line(rows, new, lens, H, KVH, page, cols, bits) for bits in (0, 32, 64)]
        for wrong, units, weight, bound, _ in got:
            assert wrong == ""
            assert units == KVH * sum(-(-n // (rows // rep)) for n in new)
            assert weight <= bound and weight == got[0][2]


def test_starts_that_do_not_ascend_and_lengths_past_the_table(line):
    for starts, lens, T in (([0, 5, 2, 7], [9, 9, 9], 7), ([-7, 2, 1 << 30], [10, 20], 5), ([3, 3, 3], [5, 5], 8),
                            ([0, 40, 0, 40, 0, 40], [100] * 5, 40), ([0, 1, 2], [2 ** 31 - 1, 50], 2)):
        for rows in (8, 16, 128):
            assert line(rows, None, lens, 8, 2, 16, 30, q_start=starts, T=T)[0] == ""


def test_the_host_takes_64_bits_for_a_long_line(line):
    """One prompt of 200000 tokens on 2 KV heads: 2.2e9 pairs of tiles and keys."""
    for rows, H, KVH in ((128, 14, 2), (16, 12, 12)):
        wrong, units, weight, bound, wide = line(rows, [200_000], [200_000], H, KVH, 16, 12_500)
        assert wrong == "" and wide and 2 ** 31 < weight <= bound
    wrong, *_, wide = line(8, [1] * 64, [600] * 64, 14, 2, 16, 40)
    assert wrong == "" and not wide


@pytest.mark.parametrize("rows,T,H,KVH,kv_len", [
    (128, 200_000, 14, 2, 0), (128, 200_000, 14, 2, 1024), (128, 200_000, 28, 4, 1024), (128, 330_000, 12, 12, 1024),
    (128, 70_000, 128, 1, 1024), (128, 95_000, 128, 1, 8192), (16, 330_000, 12, 12, 500)])
def test_more_new_tokens_than_keys(line, rows, T, H, KVH, kv_len):
    """The first tokens of a sequence see nothing; the line is no longer than the host's bound, which goes by the table."""
    wrong, units, weight, bound, wide = line(rows, [T], [kv_len], H, KVH, 16, max(1, kv_len // 16))
    assert wrong == "" and weight <= bound
    assert units == KVH * -(-T // (rows // (H // KVH)))


@pytest.mark.parametrize("seed", range(60))
def test_short_sequences_weigh_the_keys_they_see(line, seed):
    rnd = random.Random(1000 + seed)
    H, KVH = LAYOUTS[seed % len(LAYOUTS)]
    new, lens = _batch(rnd, True)
    cols = -(-max(lens + [1]) // 8)
    over = {8: 16, 16: 16, 128: 192}
    for rows in (8, 16, 128):
        tpt = rows // (H // KVH)
        if tpt == 0:
            continue
        want = KVH * sum(over[rows] + max(0, n_kv - n + min(n, t + tpt))
                         for n, n_kv in zip(new, lens) for t in range(0, n, tpt))
        for bits in (0, 32, 64):
            wrong, _, weight, bound, _ = line(rows, new, lens, H, KVH, 8, cols, bits)
            assert wrong == "" and weight == want and weight <= bound


@pytest.mark.parametrize("rows", [8, 128])
@pytest.mark.parametrize("new", [1, 20, 300])
def test_positions_up_to_the_last_that_is_accepted(line, rows, new):
    """Tables of just below 2^31 positions: a unit's weight passes 2^31."""
    top = 2 ** 31 - 8
    for lens in ([top], [top - 200, 5, top]):
        wrong, units, weight, bound, wide = line(rows, [new] * len(lens), lens, 8, 4, 8, top // 8)
        assert wrong == "" and wide and weight <= bound and units == 4 * len(lens) * -(-new // (rows // 2))
