"""GPU: the gradients of keys and values where many query heads share few key tiles, whose queries several workgroups then sum,
against 64 bits. Bounds: tests/window_ref.py."""
import pytest
import torch

from sorernn_amd import window
from tests.test_gpu_window import DEV, _bounds, _call, _inputs
from tests.test_gpu_window_more import _grads, _masked
from tests.window_ref import check, one_head, seen, window_attention as reference

pytestmark = pytest.mark.gpu
NAMES = ("o", "dq", "dk", "dv")

CASES = [
    # B, T, HQ, HKV, D, window, sinks, lens
    (1, 1, 16, 1, 64, None, 0, None),
    (1, 64, 16, 1, 128, None, 0, None),
    (1, 130, 16, 1, 64, 50, 3, None),
    (2, 513, 16, 1, 128, None, 0, None),
    (1, 700, 15, 1, 64, 300, 0, None),
    (1, 1100, 8, 1, 128, 70, 130, None),
    (1, 1500, 16, 2, 64, 333, 9, None),
    (1, 1300, 16, 2, 128, None, 0, [1, 700, 64, 535]),
    (1, 900, 12, 1, 64, 40, 5, [2, 400, 498]),
    (1, 4100, 16, 4, 128, None, 0, None),
]


@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}x{c[1]}-h{c[2]}.{c[3]}-{c[4]}-w{c[5]}.{c[6]}{'-docs' if c[7] else ''}" for c in CASES])
def test_backward(case):
    b, t, hq, hkv, d, win, sinks, lens = case
    *x, do = _inputs(b, t, hq, hkv, d, seed=11)
    leaves = [y.requires_grad_(True) for y in x]
    grads = torch.autograd.grad(_call(leaves, win, sinks, 0.11, _bounds(lens)), leaves, do)
    with torch.no_grad():
        ref = reference(*x, win, sinks, 0.11, _bounds(lens), do)
    for name, g in zip(NAMES[1:], grads):
        check(g, ref, name)
    again = torch.autograd.grad(_call(leaves, win, sinks, 0.11, _bounds(lens)), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("t, bounds", [(600, [0, 150, 333]), (600, [200, 200, 599, 599]), (300, [0, 0, 0])])
def test_bounds_as_replayed_calls_take_them(t, bounds):
    *x, do = _inputs(1, t, 16, 1, 128, seed=12)
    cu, n = torch.tensor(bounds, device=DEV), len(bounds) - 1
    o, lse = window.fwd_impl(*x, cu, 100, 3, 0.125, 0, n, True)
    grads = window.bwd_impl(*x, o, lse, do, cu, 100, 3, 0.125, 0, n)
    ref = reference(*x, 100, 3, 0.125, bounds, do)
    for name, g in zip(NAMES[1:], grads):
        check(g, ref, name)
        assert not g[:, :bounds[0]].any() and not g[:, bounds[-1]:].any()


@pytest.mark.parametrize("what, value", [("v", torch.inf), ("k", torch.nan), ("k", torch.inf), ("q", torch.nan), ("do", torch.inf)])
@pytest.mark.parametrize("t, d, win, sinks, at", [(300, 64, 40, 0, 130), (300, 128, None, 0, 70), (400, 64, 30, 5, 2)])
def test_infinities_and_nan_reach_who_sees_them(t, d, win, sinks, at, what, value):
    heads = 16
    *x, do = _inputs(1, t, heads, 1, d, seed=13)
    x = dict(zip(("q", "k", "v", "do"), (*x, do)))
    x[what][0, at, 0, 5] = value
    clean = {m: torch.where(y.isfinite(), y, 0) for m, y in x.items()}
    _, *grads = _grads((x["q"], x["k"], x["v"]), x["do"], window=win, sinks=sinks)
    places = torch.arange(t, device=DEV)
    ref = {m: torch.zeros(t, d, dtype=torch.float64, device=DEV) for m in ("dk", "dk_tol", "dv", "dv_tol")}
    want = {n: torch.zeros_like(ref[n]) for n in ("dk", "dv")}
    for h in range(heads):
        mask = seen(places, places, win, sinks) & ~((x["q"][0, :, h].double() @ x["k"][0, :, 0].double().T) == -torch.inf)
        clear = one_head(clean["q"][0, :, h], clean["k"][0, :, 0], clean["v"][0, :, 0], mask, d**-0.5, 2.0**-8, False,
                         clean["do"][0, :, h])
        for m, y in zip(("dk", "dk_tol", "dv", "dv_tol"), clear[4:]):
            ref[m] += y
        both = _masked(x["q"][0, :, h], x["k"][0, :, 0], x["v"][0, :, 0], x["do"][0, :, h], win, sinks, d**-0.5)
        for n, y in zip(("dk", "dv"), both[2:]):
            want[n] += y
    for name, g in zip(("dk", "dv"), grads[1:]):
        g, fine = g[0, :, 0], want[name].isfinite()
        assert torch.equal(g.isfinite(), fine), (name, int((g.isfinite() != fine).sum()))
        check(torch.where(fine, g, 0), {m: torch.where(fine, ref[m], 0) for m in (name, name + "_tol")}, name)


def test_captured():
    x = _inputs(1, 700, 16, 1, 64, seed=14)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _grads(x[:3], x[3], window=300, sinks=2)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _grads(x[:3], x[3], window=300, sinks=2)
    for seed in (15, 16, 17):
        for y, new in zip(x, _inputs(1, 700, 16, 1, 64, seed=seed)):
            y.copy_(new)
        graph.replay()
        got = [y.clone() for y in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, _grads(x[:3], x[3], window=300, sinks=2)))
