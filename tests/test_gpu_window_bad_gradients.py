"""GPU: a training step whose incoming gradient or keys hold infinities or NaN while the rest is healthy: what is not finite and
what is, and that such a step takes about as long as another. Bounds of the finite parts: tests/window_ref.py."""
import pytest
import torch

from tests.test_gpu_window import DEV, _inputs
from tests.test_gpu_window_more import _grads, _masked
from tests.window_ref import check, one_head, seen

pytestmark = pytest.mark.gpu


def _ms(fn):
    fn()
    best = float("inf")
    for _ in range(3):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        a.record()
        fn()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


def _all(do):
    do.fill_(torch.nan)


def _late(do):
    do[:, -9, -1, 3] = torch.nan


def _some(do):
    do[:, 50::997, 0, 7] = torch.inf


@pytest.mark.parametrize("spoil", [_all, _late, _some])
@pytest.mark.parametrize("win, sinks", [(None, 0), (1024, 4)])
@pytest.mark.parametrize("t, hq, hkv", [(3000, 4, 2), (6000, 16, 4), (1024, 16, 1)])
def test_a_bad_incoming_gradient_takes_no_longer(t, hq, hkv, win, sinks, spoil):
    """A healthy step of these sizes takes 0.2 to 0.9 ms; going over all queries of every key one by one takes 6 to 95."""
    *x, do = _inputs(1, t, hq, hkv, 128, seed=1)
    healthy = _ms(lambda: _grads(x, do, window=win, sinks=sinks))
    spoil(do)
    bad = _ms(lambda: _grads(x, do, window=win, sinks=sinks))
    print(f"{healthy:.2f} ms, {bad:.2f} ms")
    assert bad < 5 * healthy + 2, (healthy, bad)
    o, dq, dk, dv = _grads(x, do, window=win, sinks=sinks)
    assert o.isfinite().all()
    rows = ~do.isfinite().all(-1)
    assert torch.equal(dq.isfinite().all(-1), ~rows)
    rep = hq // hkv
    at = torch.arange(t, device=DEV)
    hit = (seen(at, at, win, sinks).T.float() @ rows[0].unflatten(-1, (hkv, rep)).any(-1).float()) > 0  # [T, HKV]
    assert not dk[0][hit].isfinite().any() and dk[0][~hit].isfinite().all()
    columns = ~do.isfinite()
    cols = torch.stack([(seen(at, at, win, sinks).T.float() @ columns[0, :, g * rep:(g + 1) * rep].any(1).float()) > 0
                        for g in range(hkv)], 1)
    assert torch.equal(~dv[0].isfinite(), cols)


@pytest.mark.parametrize("win, sinks", [(None, 0), (1024, 4)])
def test_an_infinite_key_takes_no_longer(win, sinks):
    """Queries of one sign there: the rows lose that key's weight and stay finite, with NaN (0 times infinity) in one column of
    their dq. Rows that share a block with it and do not see it are taken again (key by key, one row after the other, 12 to 29 ms)."""
    *x, do = _inputs(1, 6000, 16, 4, 128, seed=2)
    healthy = _ms(lambda: _grads(x, do, window=win, sinks=sinks))
    x[0][..., 5] = -x[0][..., 5].abs() - 1
    x[1][:, 40, :, 5] = torch.inf
    bad = _ms(lambda: _grads(x, do, window=win, sinks=sinks))
    print(f"{healthy:.2f} ms, {bad:.2f} ms")
    assert bad < 5 * healthy + 2, (healthy, bad)


CASES = [
    # T, heads (of one kv head), D, window, sinks, spoiled (what, token, head, column, value)
    (300, 2, 64, None, 0, [("do", 299, 1, 3, torch.nan)]),
    (300, 2, 64, None, 0, [("do", 10, 0, 3, torch.inf), ("do", 200, 1, 9, -torch.inf)]),
    (500, 16, 128, 60, 5, [("do", 499, 15, 70, torch.inf), ("do", 100, 3, 1, torch.nan)]),
    (500, 3, 128, 60, 5, [("q", 499, 2, 70, torch.inf), ("k", 130, 0, 5, torch.inf)]),
    (700, 4, 64, 50, 200, [("do", 650, 1, 33, torch.inf), ("do", 3, 0, 33, torch.inf)]),
    (400, 2, 64, None, 0, [("k", 130, 0, 5, torch.inf), ("do", 390, 0, 8, torch.inf)]),
    (400, 2, 128, 64, 0, [("v", 131, 0, 100, -torch.inf), ("do", 200, 0, 8, torch.inf)]),
]


@pytest.mark.parametrize("t, heads, d, win, sinks, spoiled", CASES, ids=[f"{c[0]}-h{c[1]}-{c[2]}-w{c[3]}.{c[4]}-{c[5][0][0]}" for c in CASES])
def test_columns(t, heads, d, win, sinks, spoiled):
    """Which entries are finite, and the values of those: as if the bad pairs' finite parts were all there was."""
    *x, do = _inputs(1, t, heads, 1, d, seed=3)
    x = dict(zip(("q", "k", "v", "do"), (*x, do)))
    for what, at, head, column, value in spoiled:
        x[what][0, at, head, column] = value
    clean = {m: torch.where(y.isfinite(), y, 0) for m, y in x.items()}
    got = dict(zip(("o", "dq", "dk", "dv"), _grads((x["q"], x["k"], x["v"]), x["do"], window=win, sinks=sinks)))
    places = torch.arange(t, device=DEV)
    keys = {m: torch.zeros(t, d, dtype=torch.float64, device=DEV) for m in ("dk", "dk_tol", "dv", "dv_tol")}
    wanted = {n: torch.zeros(t, d, dtype=torch.float64, device=DEV) for n in ("dk", "dv")}
    for h in range(heads):
        mask = seen(places, places, win, sinks) & ~((x["q"][0, :, h].double() @ x["k"][0, :, 0].double().T) == -torch.inf)
        clear = dict(zip(("o", "o_tol", "dq", "dq_tol", "dk", "dk_tol", "dv", "dv_tol"),
                         one_head(clean["q"][0, :, h], clean["k"][0, :, 0], clean["v"][0, :, 0], mask, d**-0.5, 2.0**-8, False,
                                  clean["do"][0, :, h])))
        want = dict(zip(("o", "dq", "dk", "dv"), _masked(x["q"][0, :, h], x["k"][0, :, 0], x["v"][0, :, 0], x["do"][0, :, h], win,
                                                         sinks, d**-0.5)))
        for name in ("o", "dq"):
            g, fine = got[name][0, :, h], want[name].isfinite()
            assert torch.equal(g.isfinite(), fine), (name, h, (g.isfinite() != fine).nonzero()[:4].tolist())
            check(torch.where(fine, g, 0), {m: torch.where(fine, clear[m], 0) for m in (name, name + "_tol")}, name)
        for m in keys:
            keys[m] += clear[m]
        for n in wanted:
            wanted[n] += want[n]
    for name in wanted:
        g, fine = got[name][0, :, 0], wanted[name].isfinite()
        assert torch.equal(g.isfinite(), fine), (name, (g.isfinite() != fine).nonzero()[:4].tolist())
        check(torch.where(fine, g, 0), {m: torch.where(fine, keys[m], 0) for m in (name, name + "_tol")}, name)


@pytest.mark.parametrize("t, heads, d, win, sinks, spoiled", [
    (300, 1, 64, 2, 5, [("do", 186, 0, 7, torch.inf)]),       # behind the last query that sees the tile, in its block
    (300, 2, 64, 2, 0, [("do", 130, 1, 7, torch.nan), ("q", 131, 0, 3, torch.inf)]),
    (500, 16, 64, 100, 0, [("do", 255, 3, 1, torch.inf)]),
    (700, 2, 128, 60, 130, [("do", 190, 0, 1, torch.nan), ("do", 320, 1, 2, torch.inf), ("do", 577, 1, 2, -torch.inf)]),
    (1000, 2, 64, 70, 4, [("do", 197, 0, 1, torch.nan), ("do", 256, 1, 2, torch.inf), ("q", 511, 1, 2, -torch.inf)]),
])
def test_blocks_that_reach_past_a_tile_s_queries(t, heads, d, win, sinks, spoiled):
    test_columns(t, heads, d, win, sinks, spoiled)


@pytest.mark.parametrize("t, win, heads", [(300, None, 2), (500, 200, 1), (900, 150, 16)])
def test_signs_of_values_gradients(t, win, heads):
    """An infinity of do reaches dv of every key that its query sees, with its sign; both signs make NaN."""
    *x, do = _inputs(1, t, heads, 1, 64, seed=4)
    up, down, both = t - 140, t - 70, t - 20
    do[0, up, 0, 3], do[0, down, heads - 1, 9] = torch.inf, -torch.inf
    do[0, up, 0, 20], do[0, both, 0, 20] = torch.inf, -torch.inf
    dv = _grads(x, do, window=win)[3][0, :, 0]
    at = torch.arange(t, device=DEV)
    by = {q: (at <= q) & ((at > q - win) if win else (at >= 0)) for q in (up, down, both)}
    want = torch.zeros(t, 3, device=DEV)
    want[by[up], 0] = torch.inf
    want[by[down], 1] = -torch.inf
    want[by[up], 2] = torch.inf
    want[by[both], 2] -= torch.inf
    for i, c in enumerate((3, 9, 20)):
        got = torch.where(dv[:, c].isfinite(), 0, dv[:, c].float())
        assert torch.equal(got.nan_to_num(7, 8, 9), want[:, i].nan_to_num(7, 8, 9)), c
