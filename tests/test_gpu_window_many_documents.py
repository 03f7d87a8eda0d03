"""GPU: attention's gradients where many documents with sinks are packed, so that only those longer than the window have partial
sums, against 64 bits. Bounds: tests/window_ref.py."""
import random

import pytest
import torch

from sorernn_amd import window
from tests.test_gpu_window import DEV, _bounds, _call, _inputs
from tests.test_gpu_window_more import _grads
from tests.window_ref import check, window_attention as reference

pytestmark = pytest.mark.gpu
NAMES = ("dq", "dk", "dv")


def _lens(total, docs, longest, seed):
    """`docs` lengths of one token and more that sum to `total`, one of them `longest`."""
    rng = random.Random(seed)
    share = [rng.random() ** 3 for _ in range(docs - 1)]
    left = total - longest - (docs - 1)
    lens = [1 + int(left * s / sum(share)) for s in share]
    lens[0] += total - longest - sum(lens)
    lens.insert(rng.randrange(docs), longest)
    return lens


CASES = [
    # T, HQ, HKV, D, window, sinks, documents, the longest
    (3000, 4, 2, 64, 40, 4, 30, 900),
    (3000, 2, 1, 128, 1, 4, 100, 1500),
    (2500, 2, 2, 64, 100, 130, 60, 1100),
    (2500, 8, 1, 128, 30, 1000, 60, 1200),
    (2000, 2, 1, 64, 20, 1 << 30, 80, 700),
    (4000, 2, 1, 64, 200, 33, 400, 328),
    (4000, 2, 1, 64, 200, 33, 400, 327),
    (1500, 2, 1, 128, 300, 4, 700, 200),
]


@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}-h{c[1]}.{c[2]}-{c[3]}-w{c[4]}.{c[5]}-n{c[6]}-l{c[7]}" for c in CASES])
def test_backward(case):
    t, hq, hkv, d, win, sinks, docs, longest = case
    lens = _lens(t, docs, longest, 1)
    *x, do = _inputs(1, t, hq, hkv, d, seed=1)
    leaves = [y.requires_grad_(True) for y in x]
    grads = torch.autograd.grad(_call(leaves, win, sinks, 0.11, _bounds(lens)), leaves, do)
    with torch.no_grad():
        ref = reference(*x, win, sinks, 0.11, _bounds(lens), do)
    for name, g in zip(NAMES, grads):
        check(g, ref, name)
    again = torch.autograd.grad(_call(leaves, win, sinks, 0.11, _bounds(lens)), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("bounds", [
    [0] * 60 + [1700] + [1700] * 60,            # one document, the others empty
    [0] * 60 + [800] * 60 + [1600],
    [200] + [200 + 20 * i for i in range(60)] + [1400] * 60,
    [0] * 50 + [140 * i for i in range(13)] + [1680] * 58,  # all just without far queries
    [5] * 121,
])
@pytest.mark.parametrize("win, sinks, hq", [(12, 5, 2), (40, 200, 16)])
def test_bounds_as_replayed_calls_take_them(bounds, win, sinks, hq):
    t = 1700
    *x, do = _inputs(1, t, hq, 1, 64, seed=2)
    cu, n = torch.tensor(bounds, device=DEV), len(bounds) - 1
    o, kept = window.fwd_impl(*x, cu, win, sinks, 0.125, 0, n, True)
    grads = window.bwd_impl(*x, o, kept, do, cu, win, sinks, 0.125, 0, n)
    ref = reference(*x, win, sinks, 0.125, bounds, do)
    for name, g in zip(NAMES, grads):
        check(g, ref, name)
        assert not g[:, :bounds[0]].any() and not g[:, bounds[-1]:].any()


def test_captured_with_other_documents():
    x = _inputs(1, 2000, 4, 1, 64, seed=3)
    sets = [_bounds(_lens(2000, 90, longest, seed)) for longest, seed in ((500, 1), (1800, 2), (60, 3))]
    host = torch.tensor(sets[0])
    cu = host.to(DEV)

    def step():
        return _grads(x[:3], x[3], window=25, sinks=140, cu_seqlens=cu, cu_seqlens_cpu=host)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed, bounds in enumerate(sets + sets[:1]):
        cu.copy_(torch.tensor(bounds))
        for y, new in zip(x, _inputs(1, 2000, 4, 1, 64, seed=10 + seed)):
            y.copy_(new)
        graph.replay()
        got = [y.clone() for y in out]
        torch.cuda.synchronize()
        now = torch.tensor(bounds)
        want = _grads(x[:3], x[3], window=25, sinks=140, cu_seqlens=now.to(DEV), cu_seqlens_cpu=now)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


def test_bad_values_stay_in_their_document():
    bounds = _bounds(_lens(2500, 60, 1100, 4))
    *x, do = _inputs(1, 2500, 2, 1, 64, seed=5)
    ref = reference(*x, 30, 150, 0.125, bounds, do)
    n = 30  # this document's tokens are bad, also those behind the window
    part = slice(bounds[n], bounds[n + 1])
    for y in (x[0], do):
        y[0, part] = torch.nan
    cu = torch.tensor(bounds, device=DEV)
    o, *grads = _grads(x, do, window=30, sinks=150, scale=0.125, cu_seqlens=cu)
    keep = torch.ones(2500, dtype=torch.bool, device=DEV)
    keep[part] = False
    for name, g in zip(NAMES, grads):
        assert g[:, part].isnan().all()
        check(g[:, keep], {m: y[:, keep] for m, y in ref.items()}, name)


def test_memory_of_many_documents():
    """65,536 tokens in 2,000 documents: the step's memory is what its inputs, outputs and what is kept take, and little more."""
    t, hq, hkv, d = 65536, 16, 8, 128
    lens = _lens(t, 2000, 3000, 6)
    *x, do = _inputs(1, t, hq, hkv, d, seed=7)
    bounds = torch.tensor(_bounds(lens))
    cu = bounds.to(DEV)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = _grads(x, do, window=256, sinks=4, cu_seqlens=cu, cu_seqlens_cpu=bounds)
    peak = torch.cuda.max_memory_allocated() - before
    own = sum(y.numel() * y.element_size() for y in out) + t * hq * (d // 2 + 1) * 4
    assert peak < own + 200e6, (peak, own)
