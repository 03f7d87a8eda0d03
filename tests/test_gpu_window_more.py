"""GPU: attention with a window and sinks where it can go wrong: infinities and NaN in masked places, large scores, views and
broadcast inputs, unchecked bounds, long inputs, other streams, captured and compiled steps. Bounds: tests/window_ref.py."""
import pytest
import torch

from sorernn_amd import window, window_attention
from tests.test_gpu_window import DEV, _inputs
from tests.window_ref import check, one_head, seen, window_attention as reference

pytestmark = pytest.mark.gpu


def _grads(x, do, **kw):
    leaves = [y.detach().requires_grad_(True) for y in x]
    o = window_attention(*leaves, **kw)
    return o.detach(), *torch.autograd.grad(o, leaves, do)


def _masked(q, k, v, do, win, sinks, scale):
    """One head's o, dq, dk, dv in 64 bits in which a masked pair takes part in no sum, whatever lies there."""
    q, k, v, do = (x.double() for x in (q, k, v, do))
    at = torch.arange(q.shape[0], device=DEV)
    m = seen(at, at, win, sinks)

    def dot(a, b):  # [T, L]
        return (a[:, None] * b[None]).sum(-1)

    def total(w, x, mask):  # sum over the second axis of w [A, B] x [B, D], masked
        return torch.where(mask[..., None], w[..., None] * x[None], 0).sum(1)

    s = torch.where(m, dot(q, k) * scale, -torch.inf)
    e = torch.where(m, torch.exp(s - s.amax(1, keepdim=True)), 0)
    p = e / e.sum(1, keepdim=True)
    o = total(p, v, m)
    ds = torch.where(m, p * (dot(do, v) - (do * o).sum(1, keepdim=True)), 0)
    return o, scale * total(ds, k, m), scale * total(ds.T, q, m.T), total(p.T, do, m.T)


BAD = [("v", torch.inf), ("v", torch.nan), ("k", torch.nan), ("k", torch.inf), ("q", torch.nan), ("q", -torch.inf), ("do", torch.nan),
       ("do", torch.inf)]


@pytest.mark.parametrize("what, value", BAD, ids=[f"{w}-{v}" for w, v in BAD])
@pytest.mark.parametrize("t, d, win, sinks, at", [(200, 64, 40, 3, 77), (300, 128, 64, 0, 130), (150, 64, None, 0, 149),
                                                  (400, 64, 30, 5, 2)])
def test_infinities_and_nan_reach_who_sees_them(t, d, win, sinks, at, what, value):
    *x, do = _inputs(1, t, 2, 1, d, seed=4)
    x = dict(zip(("q", "k", "v", "do"), (*x, do)))
    x[what][0, at, 0, 5] = value
    clean = {m: torch.where(y.isfinite(), y, 0) for m, y in x.items()}
    o, *grads = _grads((x["q"], x["k"], x["v"]), x["do"], window=win, sinks=sinks)
    names = ("o", "dq", "dk", "dv")
    places = torch.arange(t, device=DEV)
    ref = {m: torch.zeros(1, t, 2 if m[:2] in ("o", "o_", "dq") else 1, d, dtype=torch.float64, device=DEV)
           for n in names for m in (n, n + "_tol")}
    want = {n: torch.zeros_like(ref[n]) for n in names}
    for h in range(2):
        # a finite result depends on no bad value: it is the one of clean inputs, without keys whose score is -inf
        mask = seen(places, places, win, sinks) & ~((x["q"][0, :, h].double() @ x["k"][0, :, 0].double().T) == -torch.inf)
        clear = one_head(clean["q"][0, :, h], clean["k"][0, :, 0], clean["v"][0, :, 0], mask, d**-0.5, 2.0**-8, False,
                         clean["do"][0, :, h])
        for m, y in zip(("o", "o_tol", "dq", "dq_tol", "dk", "dk_tol", "dv", "dv_tol"), clear):
            ref[m][0, :, h if m[:2] in ("o", "o_", "dq") else 0] += y
        for n, y in zip(names, _masked(x["q"][0, :, h], x["k"][0, :, 0], x["v"][0, :, 0], x["do"][0, :, h], win, sinks, d**-0.5)):
            want[n][0, :, h if n in ("o", "dq") else 0] += y
    for name, g in zip(names, (o, *grads)):
        fine = want[name].isfinite()
        assert torch.equal(g.isfinite(), fine), (name, int((g.isfinite() != fine).sum()))
        part = {m: torch.where(fine, ref[m], 0) for m in (name, name + "_tol")}
        check(torch.where(fine, g, 0), part, name)


def test_bad_values_in_the_next_document_and_behind_the_end():
    """Rows that share tiles with another document's infinities."""
    *x, do = _inputs(1, 300, 2, 2, 64, seed=5)
    bounds = [0, 70, 130, 300]
    clean = [y.clone() for y in (*x, do)]
    for y in (*x, do):
        y[0, 70:130] = torch.nan
    cu = torch.tensor(bounds, device=DEV)
    o, *grads = _grads(x, do, window=20, sinks=2, cu_seqlens=cu)
    ref = reference(*clean[:3], 20, 2, 64**-0.5, bounds, clean[3])
    for name, g in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        assert g[0, 70:130].isnan().all()
        for part in (slice(0, 70), slice(130, 300)):
            check(g[:, part], {m: y[:, part] for m, y in ref.items()}, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_large_scores(dtype):
    """Scores in the thousands: one key takes a row; the running maximum moves at every block."""
    q, k, v, _ = _inputs(1, 500, 2, 1, 128, dtype, seed=6)
    k *= 8 * torch.linspace(0, 1, 500, device=DEV, dtype=dtype)[None, :, None, None]
    q *= 8
    for scale in (1.0, 1e-3, 30.0):
        o = window_attention(q, k, v, window=333, sinks=1, scale=scale)
        check(o, reference(q, k, v, 333, 1, scale), "o")
    zero = torch.zeros_like(q)
    o = window_attention(zero, k, v, window=100)  # equal scores
    check(o, reference(zero, k, v, 100, 0, 128**-0.5), "o")


def test_views_give_the_same_bits():
    b, t, hq, hkv, d = 2, 333, 4, 2, 64
    gen = torch.Generator(DEV).manual_seed(7)
    proj = torch.randn(b, t, (hq + 2 * hkv) * d, generator=gen, device=DEV).bfloat16()
    views = [y.unflatten(-1, (-1, d)) for y in proj.split([hq * d, hkv * d, hkv * d], -1)]
    do = torch.randn(b, hq, t, d, generator=gen, device=DEV).bfloat16().transpose(1, 2)
    want = _grads([y.contiguous() for y in views], do.contiguous(), window=50, sinks=3)
    leaf = proj.detach().requires_grad_(True)
    o = window_attention(*(y.unflatten(-1, (-1, d)) for y in leaf.split([hq * d, hkv * d, hkv * d], -1)), window=50, sinks=3)
    (dproj,) = torch.autograd.grad(o, leaf, do)
    assert torch.equal(o.detach(), want[0])
    assert torch.equal(dproj, torch.cat([g.flatten(2) for g in want[1:]], -1))
    odd = torch.randn(b * t * hkv * d + 1, generator=gen, device=DEV).bfloat16()[1:].view(b, t, hkv, d)
    head_major = [y.transpose(1, 2).contiguous().transpose(1, 2) for y in views]
    assert torch.equal(window_attention(*head_major, window=50, sinks=3), want[0])
    assert torch.equal(window_attention(views[0], odd, odd), window_attention(views[0].contiguous(), odd.clone(), odd.clone()))


def test_broadcast_keys_and_values():
    """One key head expanded over the query heads, one batch row over the batch: gradients sum."""
    q, k, v, do = _inputs(2, 130, 4, 1, 64, seed=8)
    small = [y[:1].detach().requires_grad_(True) for y in (k, v)]
    o = window_attention(q, *(y.expand(2, 130, 4, 64) for y in small), window=33, sinks=1)
    assert torch.equal(o.detach(), window_attention(q, *(y.detach().expand(2, 130, 4, 64).contiguous() for y in small), window=33, sinks=1))
    dk, dv = torch.autograd.grad(o, small, do)
    full = _grads((q, *(y.detach().expand(2, 130, 4, 64).contiguous() for y in small)), do, window=33, sinks=1)
    assert torch.equal(dk, full[2].sum((0, 2), keepdim=True)) and torch.equal(dv, full[3].sum((0, 2), keepdim=True))
    same = k[:, :1].expand(2, 130, 1, 64)  # every token the same key: stride 0 between tokens
    check(window_attention(q, same, v, window=20), reference(q, same, v, 20, 0, 64**-0.5), "o")


BOUNDS = [
    (300, [0, 200, 200]), (300, [0, 1, 200, 200, 200, 200]), (300, [70, 70, 300]), (300, [0, 0, 130, 130, 131, 131]),
    (300, [0, 0, 0]), (300, [300, 300, 300]), (1500, [0, 1200, 1300, 1300]), (1500, [130, 130, 900, 900, 900, 1500]),
    (700, [0, 650] + [650] * 200), (400, [100, 300]),
]


@pytest.mark.parametrize("t, bounds", BOUNDS, ids=[f"{t}-{'.'.join(map(str, b[:6]))}" for t, b in BOUNDS])
def test_bounds_as_replayed_calls_take_them(t, bounds):
    """Empty documents and tokens of none: zeros there, the documents' results elsewhere."""
    *x, do = _inputs(1, t, 2, 1, 64, seed=9)
    cu, n = torch.tensor(bounds, device=DEV), len(bounds) - 1
    o, lse = window.fwd_impl(*x, cu, 40, 3, 0.125, 0, n, True)
    grads = window.bwd_impl(*x, o, lse, do, cu, 40, 3, 0.125, 0, n)
    ref = reference(*x, 40, 3, 0.125, bounds, do)
    for name, g in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        check(g, ref, name)
        assert not g[:, :bounds[0]].any() and not g[:, bounds[-1]:].any()


def test_past_32_bit_offsets():
    """2.3e9 elements of q: the last tokens see only what is near them."""
    t, hq, d, win = 140001, 128, 128, 50
    gen = torch.Generator(DEV).manual_seed(10)
    q = torch.empty(1, t, hq, d, device=DEV, dtype=torch.bfloat16).normal_(generator=gen)
    do = torch.empty(1, t, hq, d, device=DEV, dtype=torch.bfloat16).normal_(generator=gen)
    k, v = (torch.empty(1, t, 1, d, device=DEV, dtype=torch.bfloat16).normal_(generator=gen) for _ in range(2))
    o, dq, dk, dv = _grads((q, k, v), do, window=win)
    end = [y[:, -300:].contiguous() for y in (q, k, v)]
    ref = reference(*end, win, 0, d**-0.5, None, do[:, -300:])
    for name, g in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        check(g[:, -200:], {m: y[:, -200:] for m, y in ref.items()}, name)


def test_gradients_against_differences():
    """The gradients' products with directions against differences of the formula's o in 64 bits."""
    *x, do = _inputs(1, 120, 2, 1, 64, seed=11)
    _, *grads = _grads(x, do, window=30, sinks=2)
    ref = reference(*x, 30, 2, 0.125, None, do)
    gen = torch.Generator(DEV).manual_seed(12)
    at = torch.arange(120, device=DEV)
    mask = seen(at, at, 30, 2)

    def loss(q, k, v):
        return sum((one_head(q[0, :, h], k[0, :, 0], v[0, :, 0], mask, 0.125, 0.0)[0] * do[0, :, h].double()).sum() for h in range(2))

    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(x[i].shape, generator=gen, device=DEV).double()
        up, down = ([y.double() + (sign * 1e-5 * way if j == i else 0) for j, y in enumerate(x)] for sign in (1, -1))
        slope = float(loss(*up) - loss(*down)) / 2e-5
        tol = float(((ref[name + "_tol"] + 2.0**-8 * (ref[name].abs() + ref[name + "_tol"])) * way.abs()).sum())
        assert abs(float((grads[i].double() * way).sum()) - slope) <= tol + 1e-6 * abs(slope), name


def test_another_stream_and_two_calls_at_once():
    *x, do = _inputs(2, 700, 4, 2, 64, seed=13)
    want = _grads(x, do, window=90, sinks=4)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(_grads(x, do, window=90, sinks=4))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_captured_steps():
    """Forward and backward in two graphs on one pool with other inputs and documents at every replay, eager work between."""
    static = [y.requires_grad_(True) for y in _inputs(1, 600, 2, 1, 64, seed=14)[:3]]
    do = _inputs(1, 600, 2, 1, 64, seed=14)[3]
    cu_host = torch.tensor([0, 300, 600])
    cu = cu_host.to(DEV)

    def step(win):
        o = window_attention(*static, window=win, sinks=2, cu_seqlens=cu, cu_seqlens_cpu=cu_host)
        return [o.detach(), *torch.autograd.grad(o, static, do)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(40), step(90)
    torch.cuda.current_stream().wait_stream(s)
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for win in (40, 90):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            outs.append(step(win))
    for seed, bounds in ((20, [0, 300, 600]), (21, [0, 599, 600]), (22, [0, 64, 600])):
        fresh = _inputs(1, 600, 2, 1, 64, seed=seed)
        with torch.no_grad():
            for y, z in zip((*static, do), fresh):
                y.copy_(z)
            cu.copy_(torch.tensor(bounds))
        for graph, out, win in zip(graphs, outs, (40, 90)):
            graph.replay()
            torch.cuda.synchronize()
            got = [y.clone() for y in out]
            want = _grads(fresh[:3], fresh[3], window=win, sinks=2, cu_seqlens=torch.tensor(bounds, device=DEV))
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (seed, win)


def test_compiled_step():
    *x, do = _inputs(1, 500, 4, 2, 64, seed=15)
    cu = torch.tensor([0, 200, 500], device=DEV)

    def fn(q, k, v):
        return window_attention(q * 1.0, k, v, window=64, sinks=2, cu_seqlens=cu)

    leaves = [y.requires_grad_(True) for y in x]
    got = torch.compile(fn, fullgraph=True)(*leaves)
    want = fn(*leaves)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, do), torch.autograd.grad(want, leaves, do)))


def test_no_tokens_and_unused_outputs():
    q, k, v, _ = _inputs(2, 3, 2, 1, 64)
    empty = [y[:, :0].detach().requires_grad_(True) for y in (q, k, v)]
    o = window_attention(*empty)
    assert o.shape == (2, 0, 2, 64)
    assert all(g.shape == y.shape for g, y in zip(torch.autograd.grad(o.sum(), empty), empty))
    # one leaf alone; a second derivative is refused
    leaf = q.detach().requires_grad_(True)
    o = window_attention(leaf, k, v)
    (g,) = torch.autograd.grad(o.float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_int32_bounds_and_their_check_without_a_host_copy():
    *x, do = _inputs(1, 300, 2, 1, 64, seed=16)
    bounds = [0, 5, 170, 300]
    want = _grads(x, do, window=40, sinks=1, cu_seqlens=torch.tensor(bounds, device=DEV))
    got = _grads(x, do, window=40, sinks=1, cu_seqlens=torch.tensor(bounds, device=DEV, dtype=torch.int32))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_nothing_but_nan():
    """A diverged step ends as soon as another: rows that see a NaN are not computed again."""
    x = [torch.full_like(y, torch.nan) for y in _inputs(1, 3000, 4, 2, 128)]
    out = _grads(x[:3], x[3])
    torch.cuda.synchronize()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    out = _grads(x[:3], x[3])
    b.record()
    torch.cuda.synchronize()
    assert all(y.isnan().all() for y in out)
    assert a.elapsed_time(b) < 50


def test_batched_gradients():
    *x, do = _inputs(1, 90, 2, 1, 64, seed=17)
    leaves = [y.requires_grad_(True) for y in x]
    o = window_attention(*leaves, window=20)
    ups = torch.stack([do, 2 * do])
    got = torch.autograd.grad(o, leaves, ups, is_grads_batched=True, retain_graph=True)
    for i in range(2):
        want = torch.autograd.grad(o, leaves, ups[i], retain_graph=True)
        assert all(torch.equal(a[i], b) for a, b in zip(got, want))
