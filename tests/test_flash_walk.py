"""CPU: which rows, keys and pieces the attention kernels' workgroups take, for bounds of every kind.

``gdn_flash_walk.h``, which the kernels include, is compiled for the host (``flash_walk.cpp``) and compared with brute force.
"""
import ctypes
import itertools
import os
import random
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
FAR = 1 << 29


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("walk") / "walk.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wall", "-Wno-unknown-pragmas", "-o", out,
                    os.path.join(HERE, "flash_walk.cpp")], check=True)
    lib = ctypes.CDLL(out)
    lib.flash_tiles.restype = lib.flash_jobs.restype = ctypes.c_int64
    return lib


def _tiles(lib, cu, tokens, mul, rows):
    room = tokens * mul // rows + len(cu) + 4
    out = np.zeros(4 * room, np.int64)
    bounds = np.array(cu, np.int64)
    n = lib.flash_tiles(bounds.ctypes.data_as(ctypes.c_void_p), ctypes.c_int64(len(cu) - 1), ctypes.c_int64(tokens), mul, rows,
                        out.ctypes.data_as(ctypes.c_void_p), ctypes.c_int64(room))
    assert n >= 0, (cu, tokens, mul, rows, n)
    return out[:4 * n].reshape(n, 4).tolist()


def _rows(lib, cu, tokens, mul, rows):
    """(first row, end, sequence) of every tile that has any, in rows of the flat axis; nothing outside it."""
    got = []
    for start, length, num, tile in _tiles(lib, cu, tokens, mul, rows):
        lo, hi = tile * rows, min((tile + 1) * rows, length * mul)
        if lo < hi:
            assert 0 <= start and start + length <= tokens
            got.append((start * mul + lo, start * mul + hi, num))
    return got


def _check_tiles(lib, cu, tokens, mul, rows):
    owner = [-1] * tokens
    for n, (a, e) in enumerate(zip(cu[:-1], cu[1:])):
        owner[a:e] = [n] * (e - a)
    seen = [None] * (tokens * mul)
    for lo, hi, num in _rows(lib, cu, tokens, mul, rows):
        for r in range(lo, hi):
            assert seen[r] is None, (cu, tokens, mul, rows, r)
            seen[r] = num
    assert seen == [owner[r // mul] for r in range(tokens * mul)], (cu, tokens, mul, rows)


def test_every_row_is_in_one_tile(lib):
    for tokens in (1, 2, 5):
        for n in (1, 2, 3):
            for cu in itertools.combinations_with_replacement(range(tokens + 1), n + 1):
                for mul, rows in ((1, 2), (3, 4), (2, 1)):
                    _check_tiles(lib, list(cu), tokens, mul, rows)
    rng = random.Random(1)
    for _ in range(60):
        tokens = rng.randint(1, 900)
        cu = sorted(rng.randint(0, tokens) for _ in range(rng.choice([2, 3, 9, 62, 63, 64, 65, 200])))
        _check_tiles(lib, cu, tokens, rng.choice([1, 2, 5, 16]), rng.choice([32, 128, 256]))


def test_bounds_out_of_order_lead_nowhere_outside(lib):
    rng = random.Random(2)
    for _ in range(300):
        tokens = rng.randint(1, 300)
        cu = [rng.choice([-5, 0, tokens, tokens + 9, 1 << 60, -(1 << 60), rng.randint(0, tokens)]) for _ in range(rng.randint(2, 130))]
        for mul, rows in ((1, 128), (4, 32)):
            _rows(lib, cu, tokens, mul, rows)


@pytest.mark.parametrize("hkv", [1, 2, 3, 4, 6, 8, 12, 16])
def test_every_job_is_taken_once(lib, hkv):
    for rep, tiles in itertools.product((1, 3), (1, 2, 7, 8, 33)):
        room = hkv * rep * (tiles + 8) * 8
        out = np.zeros(3 * room, np.int64)
        n = lib.flash_jobs(hkv, rep, ctypes.c_int64(tiles), out.ctypes.data_as(ctypes.c_void_p), ctypes.c_int64(room))
        assert n > 0 and n % 8 == 0
        jobs = [tuple(x) for x in out[:3 * n].reshape(n, 3).tolist() if x[0] >= 0]
        assert sorted(jobs) == sorted(itertools.product(range(hkv), range(rep), range(tiles)))
        where = {}
        for i, x in enumerate(out[:3 * n].reshape(n, 3).tolist()):
            where.setdefault(x[0], set()).add(i % 8)
        assert all(len(x) <= max(1, 8 // hkv if 8 % hkv == 0 else 8) for h, x in where.items() if h >= 0)


def _sees(q, k, window, sinks):
    return k <= q and (q - k < window or k < sinks)


def test_blocks_hold_what_is_seen(lib):
    rng = random.Random(3)
    for _ in range(400):
        first = rng.randint(-5, 400)
        last = first + rng.randint(0, 130)
        window, sinks = rng.choice([1, 2, 31, 64, 65, 200, FAR]), rng.choice([0, 1, 4, 63, 64, 65, 300, FAR])
        if window == FAR:
            sinks = 0
        size = rng.choice([32, 64])
        out = np.zeros(64, np.int32)
        n = lib.flash_blocks(size, first, last, window, sinks, out.ctypes.data_as(ctypes.c_void_p))
        got = out[:n].tolist()
        assert len(set(got)) == n and got == sorted(got)
        need = {k // size for q in range(first, last + 1) for k in range(0, q + 1) if _sees(q, k, window, sinks)}
        assert need <= set(got)
        assert all(0 <= b <= max(last, 0) // size for b in got)
        for b in got + [max(got, default=0) + 1]:
            k0, k1 = b * size, b * size + size - 1
            pairs = [_sees(q, k, window, sinks) for q in (range(first, last + 1)) for k in range(k0, k1 + 1)]
            bits = lib.flash_sees(first, last, k0, k1, window, sinks)
            assert not bits & 1 or all(pairs)
            assert not bits & 2 or not any(pairs)


def test_every_query_of_a_sink_is_summed_once(lib):
    """Near queries of a key tile and the pieces of the far ones, as the key gradients' kernel takes them."""
    rng = random.Random(4)
    for _ in range(60):
        tokens = rng.randint(1, 2500)
        cu = sorted(rng.randint(0, tokens) for _ in range(rng.randint(2, 6)))
        window, sinks, far = rng.choice([1, 30, 200, 700]), rng.choice([1, 5, 128, 129, 300]), rng.choice([256, 512])
        pieces = _tiles(lib, cu, tokens, 1, far)
        for num, (a, e) in enumerate(zip(cu[:-1], cu[1:])):
            length = e - a
            mine = [(slot, tile) for slot, (start, ln, s, tile) in enumerate(pieces) if s == num and ln and tile * far < ln]
            # a sequence's pieces lie one behind the other from b0 / far + num + 1 on
            assert [slot for slot, _ in mine] == [a // far + num + 1 + i for i in range(-(-length // far))]
            for tile in range(-(-min(sinks, length) // 128)):
                end = lib.flash_near_end(tile, window, length)
                count = [1 if tile * 128 <= q < end else 0 for q in range(length)]
                for _, piece in mine:
                    for q in range(max(end, piece * far), min(length, (piece + 1) * far)):
                        count[q] += 1
                assert all(count[q] == (1 if q >= tile * 128 else 0) for q in range(length))
                assert not any(_sees(q, k, window, 0) for q in range(end, min(length, end + 40))
                               for k in (tile * 128, min(tile * 128 + 127, length - 1)))
