"""CPU: which tokens the chunked decay linear attention walks, for documents' bounds of every kind.

``gdn_linear_walk.h``, which the kernels include, is compiled for the host (``linear_walk.cpp``) and run over segments.
"""
import ctypes
import itertools
import os
import random
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("walk") / "walk.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-Wall", "-Wno-unknown-pragmas", "-o", out,
                    os.path.join(HERE, "linear_walk.cpp")], check=True)
    return ctypes.CDLL(out)


def _chunks(lib, cu, tokens, rev, lo, hi, seq=0):
    most = tokens + 2
    out, ends = np.zeros(5 * most, np.int32), np.zeros(2, np.int32)
    bounds = None if cu is None else np.array(cu, np.int64)
    n = len(cu) - 1 if cu is not None else tokens // seq
    count = lib.linear_walk(None if cu is None else bounds.ctypes.data_as(ctypes.c_void_p), n, tokens, seq, int(rev), lo, hi,
                            out.ctypes.data_as(ctypes.c_void_p), most, ends.ctypes.data_as(ctypes.c_void_p))
    assert 0 <= count < most, (cu, tokens, rev, lo, hi, count)
    chunks = out[:5 * count].reshape(count, 5).tolist()
    first, last = ends.tolist()
    assert lo <= min(first, last) and max(first, last) <= hi, (cu, tokens, rev, lo, hi, first, last)
    at = first  # they cover what lies between their ends
    for t, ln, *_ in chunks:
        assert (t + ln if rev else t) == at, (cu, tokens, rev, lo, hi, first, last, t, ln)
        at = t if rev else t + ln
    assert at == last
    return chunks


def _span(lib, cu, tokens, lo, hi, seq=0):
    out = np.zeros(4, np.int32)
    bounds = None if cu is None else np.array(cu, np.int64)
    n = len(cu) - 1 if cu is not None else tokens // seq
    assert lib.linear_span(None if cu is None else bounds.ctypes.data_as(ctypes.c_void_p), n, tokens, seq, lo, hi,
                           out.ctypes.data_as(ctypes.c_void_p)) == 0, (cu, tokens, lo, hi)
    return out.tolist()


def _check(lib, cu, tokens, length, seq=0):
    """Every token of a document once, in its document, the documents' ends where they are, and no other token."""
    docs = [(p, e) for p, e in zip(cu[:-1], cu[1:])] if cu is not None else [(i, i + seq) for i in range(0, tokens, seq)]
    for rev in (False, True):
        doc_of = {}
        for lo in range(0, tokens, length):
            hi = min(lo + length, tokens)
            chunks = _chunks(lib, cu, tokens, rev, lo, hi, seq)
            at = hi if rev else lo
            for i, (t, ln, n, fresh, done) in enumerate(chunks):
                what = (cu, tokens, length, "rev" if rev else "fwd", lo, (t, ln, n, fresh, done))
                assert lo <= t and t + ln <= hi and 0 < ln <= 64, what
                assert (t + ln <= at) if rev else (t >= at), what
                at = t if rev else t + ln
                p, e = docs[n]
                assert p <= t and t + ln <= e, what
                assert fresh == (t + ln == e if rev else t == p), what
                assert done == (t == p if rev else t + ln == e), what
                # what is not fresh goes on from the chunk before, or is the first and comes from the segment's border
                assert fresh or i or (t + ln == hi if rev else t == lo), what
                for x in range(t, t + ln):
                    assert x not in doc_of, what
                    doc_of[x] = n
        assert doc_of == {x: n for n, (p, e) in enumerate(docs) for x in range(p, e)}, (cu, tokens, length, rev)
    for lo in range(0, tokens, length):  # what the gate's gradient takes of a segment
        hi = min(lo + length, tokens)
        t0, t1, first, last = _span(lib, cu, tokens, lo, hi, seq)
        inside = [x for x in range(lo, hi) if x in doc_of]
        what = (cu, tokens, lo, hi, t0, t1, first, last)
        if not inside:
            assert t0 >= t1, what
        else:
            assert (t0, t1, first, last) == (inside[0], inside[-1] + 1, doc_of[inside[0]], doc_of[inside[-1]]), what


@pytest.mark.parametrize("cu, tokens", [
    ([0, 200, 200], 300),            # an empty document at the end and tokens behind it
    ([0, 300, 650, 650], 700),
    ([0, 50, 50], 100),
    ([50, 50, 100], 100),            # an empty one at the beginning and tokens before it
    ([50, 50, 50, 90, 90, 90], 100),
    ([0, 0, 0], 100),                # nothing but empty ones
    ([100, 100, 100], 100),
    ([40, 40], 100),
    ([0, 64, 64, 64, 699], 700),
    ([0] + [200] * 300, 300),
    ([0] * 300 + [200], 300),
    ([0, 100] + [200] * 5000, 300),
])
def test_empty_documents_and_loose_tokens(lib, cu, tokens):
    for length in (128, 192, tokens):
        _check(lib, cu, tokens, length)


def test_all_small_ascending_bounds(lib):
    marks = [0, 1, 63, 64, 65, 128, 130, 200, 256, 260]
    for n in (1, 2, 3):
        for cu in itertools.combinations_with_replacement(marks, n + 1):
            for length in (128, 260):
                _check(lib, list(cu), 260, length)


def test_random_ascending_bounds(lib):
    rng = random.Random(0)
    for _ in range(400):
        tokens = rng.choice([70, 385, 700, 1500])
        n = rng.choice([1, 5, 63, 64, 65, 200])
        cu = sorted(rng.choice([rng.randint(0, tokens), rng.randint(0, 5) * tokens // 5]) for _ in range(n + 1))
        _check(lib, cu, tokens, rng.choice([128, 192, 256, tokens]))


def test_sequences_of_one_length(lib):
    for tokens, seq in ((8 * 50, 50), (3 * 700, 700), (64, 64), (5, 1)):
        for length in (128, tokens):
            _check(lib, None, tokens, length, seq)


def test_any_bounds_stay_inside(lib):
    """Unchecked bounds: no token outside the segment, none twice, and the first chunk is not taken for the rest of a
    document unless it lies at a border inside the token axis, where a state is kept."""
    rng = random.Random(1)
    for _ in range(3000):
        tokens = rng.choice([70, 300, 700])
        cu = [rng.choice([rng.randint(-50, tokens + 50), 0, tokens, -2**62, 2**62]) for _ in range(rng.choice([2, 3, 5, 90]))]
        length = rng.choice([128, tokens])
        for rev in (False, True):
            for lo in range(0, tokens, length):
                hi = min(lo + length, tokens)
                at = hi if rev else lo
                for i, (t, ln, n, fresh, done) in enumerate(_chunks(lib, cu, tokens, rev, lo, hi)):
                    what = (cu, tokens, length, rev, lo, (t, ln, n, fresh, done))
                    assert lo <= t and 0 < ln <= 64 and t + ln <= hi and 0 <= n < len(cu) - 1, what
                    assert (t + ln <= at) if rev else (t >= at), what
                    at = t if rev else t + ln
                    if i == 0 and not fresh:
                        assert (hi < tokens and t + ln == hi) if rev else (lo > 0 and t == lo), what
                t0, t1, first, last = _span(lib, cu, tokens, lo, hi)
                assert 0 <= first < len(cu) - 1 and 0 <= last < len(cu) - 1 and t0 >= lo and t1 <= hi
