"""CPU: the pieces of far queries and the slots of their sums in the key gradients of attention's sinks, by number and by start.

``gdn_flash_walk.h``, which the kernels include, is compiled for the host (``far_walk.cpp``) and compared with brute force.
"""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

from sorernn_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))
I64, P = ctypes.c_int64, ctypes.c_void_p


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("far") / "far.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wall", "-Wno-unknown-pragmas", "-o", out,
                    os.path.join(HERE, "far_walk.cpp")], check=True)
    lib = ctypes.CDLL(out)
    lib.far_jobs.restype = lib.near_slots.restype = I64
    return lib


def _bounds(cu):
    return None if cu is None else np.array(cu, np.int64)


def _jobs(lib, cu, n, rows, tokens, far, tiles, start, reach, count):
    out = np.zeros((count, 8), np.int64)
    b = _bounds(cu)
    bad = lib.far_jobs(None if b is None else b.ctypes.data_as(P), I64(n), I64(rows), I64(tokens), far, tiles, start, reach, I64(count),
                       out.ctypes.data_as(P))
    assert bad == 0
    return out.tolist()


def _near(lib, cu, n, tokens, far, tiles, start, reach, count):
    out = np.zeros((count, 6), np.int64)
    b = _bounds(cu)
    bad = lib.near_slots(None if b is None else b.ctypes.data_as(P), I64(n), I64(tokens), far, tiles, start, reach, I64(count),
                         out.ctypes.data_as(P))
    assert bad == 0
    return out.tolist()


def _check(lib, cu, rows, tokens, window, sinks, by_start):
    """Every query behind a tile of sinks' near ones is in one piece, pieces' and tiles' slots are their own, and the sums are
    looked for where they are."""
    reach, tiles = window + 128, -(-min(sinks, tokens) // 128)
    far, start = 256 * tiles, lib.far_start(reach, tiles) if by_start else 0
    n = rows if cu is None else len(cu) - 1
    if by_start:
        count = near_count = tokens // start
    else:
        count = (tokens // far + n + 2 if cu else rows * -(-tokens // far)) * tiles
        near_count = n * tiles
    jobs = _jobs(lib, cu, n, rows, tokens, far, tiles, start, reach, count)
    first = lib.far_first(start, reach)
    spans = [(i, 0, tokens) for i in range(rows)] if cu is None else [(0, s, e - s) for s, e in zip(cu[:-1], cu[1:])]
    near = _near(lib, cu, n, tokens, far, tiles, start, reach, near_count)
    slots = {}
    for x, (row, begin, length, num, tile, slot) in enumerate(near):
        if tile >= 0:
            assert slot == x and (row, begin, length) == spans[num]
            slots[num, tile] = x
    work = {}
    for t, (row, begin, length, num, piece, tile, at, step) in enumerate(jobs):
        if tile < 0:
            continue
        num = row if cu is None else num
        assert (row, begin, length) == spans[num]
        assert at + piece * step == t  # where the last kernel looks for this piece of this tile
        assert (num, tile, piece) not in work
        work[num, tile, piece] = t
    for num, (_, _, length) in enumerate(spans):
        for tile in range(tiles):
            near_end = min(length, tile * 128 + 127 + window)
            if near_end >= length:
                continue
            assert (num, tile) in slots
            got = []
            for (m, s, piece) in work:
                if (m, s) == (num, tile):
                    got += range(max(near_end, first + piece * far), min(length, first + (piece + 1) * far))
            assert sorted(got) == list(range(near_end, length)), (num, tile)
            pieces = range((near_end - first) // far, (length - 1 - first) // far + 1)
            assert all((num, tile, m) in work for m in pieces)
    return tiles, start


def test_by_number(lib):
    rng = random.Random(1)
    for _ in range(40):
        tokens = rng.randint(130, 3000)
        cu = sorted(rng.randint(0, tokens) for _ in range(rng.randint(2, 6)))
        _check(lib, cu, 1, tokens, rng.choice([1, 30, 200, 700]), rng.choice([1, 5, 128, 129, 300, 4000]), False)
        _check(lib, None, rng.randint(1, 3), tokens, rng.choice([1, 30, 200]), rng.choice([1, 129, 300]), False)


def test_by_start(lib):
    rng = random.Random(2)
    for _ in range(80):
        tokens = rng.randint(130, 4000)
        window = rng.choice([1, 30, 200, 700])
        lens, left = [], tokens
        while left > 0:  # some with far queries, some that just have none, empty ones
            m = min(left, rng.choice([0, 1, 50, window + 127, window + 128, window + 300, window + 900]))
            lens.append(m)
            left -= m
            if len(lens) > 200:
                break
        begin = rng.choice([0, 0, rng.randint(0, left)]) if left else 0
        cu = [begin]
        for m in lens:
            cu.append(cu[-1] + m)
        _check(lib, cu, 1, tokens, window, rng.choice([1, 5, 128, 129, 300, 1000, 4000]), True)


def test_by_start_holds_every_length(lib):
    """A sequence's tiles times pieces fit between its start and the next one's: brute force over lengths."""
    for window in (1, 2, 50, 128, 200, 256, 1024, 5000):
        reach = window + 128
        for tiles in (1, 2, 3, 8, 40):
            start = lib.far_start(reach, tiles)
            assert 128 <= start <= 256
            for length in range(1, 3 * 256 * tiles + 2 * reach, 1 if tiles < 4 else 7):
                n = lib.far_tiles(reach, tiles, length)
                assert n == (min(tiles, 1 + (length - reach) // 128) if length >= reach else 0)
                if n:
                    assert n * (1 + (length - reach) // (256 * tiles)) <= length // start, (window, tiles, length)


def test_bounds_out_of_order_lead_nowhere_outside(lib):
    rng = random.Random(3)
    for _ in range(200):
        tokens = rng.randint(140, 3000)
        cu = [rng.choice([-5, 0, tokens, tokens + 9, 1 << 60, -(1 << 60), rng.randint(0, tokens)]) for _ in range(rng.randint(2, 130))]
        window, tiles = rng.choice([1, 100]), rng.choice([1, 3])
        start = lib.far_start(window + 128, tiles)
        count = tokens // start
        for row, begin, length, num, piece, tile, at, step in _jobs(lib, cu, len(cu) - 1, 1, tokens, 256 * tiles, tiles, start, window + 128, count):
            if tile >= 0:
                assert 0 <= begin and begin + length <= tokens and 0 <= at < count and 0 <= piece and at + piece * step < count
        for row, begin, length, num, tile, slot in _near(lib, cu, len(cu) - 1, tokens, 256 * tiles, tiles, start, window + 128, count):
            if tile >= 0:
                assert 0 <= begin and begin + length <= tokens and 0 <= slot < count


def _size(tokens, docs, hkv, window, sinks, d=128, hq=16):
    return _lib.load().gdn_window_attn_bwd_workspace_size(1, tokens, hq, hkv, d, docs, window, sinks, 1)


def test_workspace_of_many_documents():
    """The sinks' sums take what documents with far queries can need, however many documents there are."""
    delta = 65536 * 16 * 4
    for docs in (600, 2000, 4000, 60000):
        assert _size(65536, docs, 8, 256, 4) - delta < 150e6
        assert _size(65536, docs, 8, 1024, 4) - delta < 150e6
    assert _size(5000, 2500, 8, 1024, 4) < 20e6
    # at most 4.5 rows of dk and dv in fp32 for each key and kv head, whatever the sinks, the window and the documents are
    for tokens in (129, 1000, 8192, 131072):
        for docs in (1, 2, 7, 60, 2000, 100000):
            if docs > tokens:
                continue
            for window in (1, 64, 256, 1000):
                for sinks in (1, 4, 32, 33, 129, 1024, 100000, 1 << 30):
                    share = 16 * tokens * 8 * 2 * 128 * 4 if docs * 128 < tokens else 0  # near sums of shared tiles, where tiles are few
                    rest = _size(tokens, docs, 8, window, sinks) - tokens * 16 * 4 - 255
                    assert rest <= 4.5 * (tokens + 512) * 8 * 2 * 128 * 4 + share, (tokens, docs, window, sinks)
