"""GPU: the paged cache where it can go wrong: bad pages and lengths, garbage behind the sequences, infinities and NaN in masked
places, large caches, shared pages, padded batches, captured calls, other streams. Bounds: tests/window_ref.py, and
tests/test_gpu_paged.py for appended rows."""
import pytest
import torch

from sorernn_amd import paged_attention, paged_kv_append
from tests.test_gpu_paged import DEV, _cache, _case, _attend, CASES
from tests.window_ref import check, gather, paged_attention as reference

pytestmark = pytest.mark.gpu


def _ref(x):
    q, kc, vc, table, lengths, win, sinks, words, bounds = x
    return reference(q, kc, vc, table, lengths, win, sinks, q.shape[-1] ** -0.5, words, bounds)


@pytest.mark.parametrize("value", [torch.nan, torch.inf])
@pytest.mark.parametrize("i", [1, 2, 4, 6, 7, 10, 12, 13, 15])
def test_garbage_behind_the_sequences(i, value):
    """Rows that no sequence has filled hold NaN: the last pages' rests and every other page."""
    x = list(_case(CASES[i], torch.bfloat16, seed=1))
    q, kc, vc, table, lengths = x[:5]
    page = kc.shape[2]
    clean = _ref(x)
    used = torch.zeros(kc.shape[0], page, dtype=torch.bool, device=DEV)
    for n, length in enumerate(lengths.tolist()):
        for s in range(length):
            used[table[n, s // page], s % page] = True
    for c in (kc, vc):
        c.masked_fill_(~used[:, None, :, None], value)
    check(_attend(*x), clean, "o")


@pytest.mark.parametrize("bad", [-1, -(2**31), 2**31 - 1, 10**6])
@pytest.mark.parametrize("i", [2, 4, 6, 8, 10, 13, 15])
def test_pages_that_the_cache_does_not_have(i, bad):
    """Their keys are not seen, wherever they stand, and what is behind a sequence's end does not matter."""
    x = list(_case(CASES[i], torch.float16, seed=2))
    table, lengths, page = x[3].clone(), x[4], x[1].shape[2]
    for n, length in enumerate(lengths.tolist()):
        whole = -(-length // page)
        table[n, whole:] = bad
        for p in {0, whole // 2, max(whole - 2, 0)} if whole > 2 else ():
            table[n, p] = bad
    x[3] = table
    check(_attend(*x), _ref(x), "o")


def test_a_sequence_without_any_page():
    x = list(_case(CASES[2], torch.bfloat16, seed=3))
    x[3] = x[3].clone()
    x[3][1] = -1
    o = _attend(*x)
    check(o, _ref(x), "o")
    assert not o[1].any()


@pytest.mark.parametrize("lengths", [[-5, 10**9, 40], [-(2**62), 2**62, 0]])
def test_lengths_out_of_range(lengths):
    """A length counts as at most what the row of the table holds; nothing is appended to such a sequence."""
    gen = torch.Generator(DEV).manual_seed(4)
    kc, vc, table = _cache(3, 64, 2, 64, 16, torch.bfloat16, gen)
    q, k, v = (torch.randn(3, 5, h, 64, generator=gen, device=DEV).bfloat16() for h in (4, 2, 2))
    lens = torch.tensor(lengths, device=DEV)
    k0, v0 = kc.clone(), vc.clone()
    paged_kv_append(k, v, kc, vc, table, lens, rot_dim=0)
    for n, length in enumerate(lengths):
        if 5 <= length <= 64:
            for t in range(5):
                s = length - 5 + t
                k0[table[n, s // 16], :, s % 16] = k[n, t]
                v0[table[n, s // 16], :, s % 16] = v[n, t]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    o = paged_attention(q, kc, vc, table, lens)
    check(o, reference(q, kc, vc, table, lens.clamp(0, 64), None, 0, 0.125), "o")


BAD = [("v", torch.inf), ("v", torch.nan), ("k", torch.nan), ("q", torch.nan)]


@pytest.mark.parametrize("what, value", BAD, ids=[f"{w}-{v}" for w, v in BAD])
@pytest.mark.parametrize("i, at", [(4, 1950), (4, 1), (6, 290), (7, 880), (8, 690), (10, 350), (11, 1350), (11, 2), (13, 3), (5, 2980)])
def test_infinities_and_nan_reach_who_sees_them(i, at, what, value):
    x = list(_case(CASES[i], torch.bfloat16, seed=5))
    q, kc, vc, table, lengths, win, sinks, words, bounds = x
    clean = _ref(x)
    page, hkv = kc.shape[2], kc.shape[1]
    rep = q.shape[2] // hkv
    count = (bounds[1] if bounds else q.shape[1])
    base = int(lengths[0]) - count
    if what == "q":
        q[0, count // 2, 0, 3] = value
        touched = torch.zeros(count, dtype=torch.bool)
        touched[count // 2] = True
        heads = slice(0, 1)
    else:
        (kc if what == "k" else vc)[table[0, at // page], 0, at % page, 3] = value
        touched = torch.zeros(count, dtype=torch.bool)
        for t in range(count):
            word = None if words is None else int(words[0, t]) & ((1 << count) - 1)
            place = base + t if word is None else base + bin(word).count("1") - 1
            if word is not None and at >= base:
                touched[t] = bool(word >> (at - base) & 1)
            else:
                touched[t] = at <= place and (win is None or place - at < win or at < sinks)
        heads = slice(0, rep)
    o = _attend(*x)
    rows = touched.nonzero()[:, 0].to(DEV)
    got = o[0, :count][:, heads][rows]
    bad = got[..., 3] if what == "v" else got
    assert not bad.isfinite().any()
    rest = o.clone()
    ref = {m: y.clone() for m, y in clean.items()}
    for y in (rest, *ref.values()):
        part = y[0, :count]
        keep = part[:, heads][rows].clone()
        keep[..., 3 if what == "v" else slice(None)] = 0
        part[rows[:, None], torch.arange(part.shape[1], device=DEV)[heads]] = keep
    check(rest, ref, "o")


def test_large_scores():
    for i in (2, 10):
        x = list(_case(CASES[i], torch.bfloat16, seed=6))
        x[1] *= 10 * torch.linspace(0, 1, x[1].shape[0], device=DEV)[:, None, None, None].bfloat16()
        x[0] *= 10
        check(_attend(*x), _ref(x), "o")


@pytest.mark.parametrize("t", [1, 40])
def test_past_32_bit_offsets(t):
    """2.3e9 elements a cache, the sequences' pages at both ends of it."""
    pages, hkv, page, d = 70000, 4, 64, 128
    kc, vc = (torch.zeros(pages, hkv, page, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    gen = torch.Generator(DEV).manual_seed(7)
    table = torch.tensor([[69999, 0, 69998, 35000], [1, 69997, 40000, 2]], dtype=torch.int32, device=DEV)
    for p in table.flatten().tolist():
        for c in (kc, vc):
            c[p] = torch.randn(hkv, page, d, generator=gen, device=DEV).bfloat16()
    q, k, v = (torch.randn(2, t, h, d, generator=gen, device=DEV).bfloat16() for h in (8, hkv, hkv))
    lengths = torch.tensor([170, 256], device=DEV)
    paged_kv_append(k, v, kc, vc, table, lengths, rot_dim=0)
    for n in range(2):
        assert torch.equal(gather(vc, table[n], int(lengths[n]))[-t:], v[n])
        assert torch.equal(gather(kc, table[n], int(lengths[n]))[-t:], k[n])
    check(paged_attention(q, kc, vc, table, lengths), reference(q, kc, vc, table, lengths, None, 0, d**-0.5), "o")


def test_shared_pages():
    """Sequences that share a prefix's pages, and one page named twice by a sequence."""
    gen = torch.Generator(DEV).manual_seed(8)
    kc, vc, table = _cache(3, 200, 2, 64, 16, torch.bfloat16, gen)
    table[1, :6] = table[0, :6]
    table[2, 3] = table[2, 1]
    q = torch.randn(3, 2, 4, 64, generator=gen, device=DEV).bfloat16()
    lengths = torch.tensor([200, 130, 77], device=DEV)
    check(paged_attention(q, kc, vc, table, lengths), reference(q, kc, vc, table, lengths, None, 0, 0.125), "o")


def test_append_leaves_the_rest_and_pads_in_front():
    """A padded batch: tokens before a sequence's first are not written; bad pages neither; other rows keep their bits."""
    gen = torch.Generator(DEV).manual_seed(9)
    kc, vc, table = _cache(4, 96, 3, 128, 32, torch.float16, gen, spare=5)
    table[2, 1] = -7
    table[3, 0] = 10**6
    k, v, q = (torch.randn(4, 50, h, 128, generator=gen, device=DEV).half() for h in (3, 3, 6))
    lengths = torch.tensor([10, 50, 60, 33], device=DEV)
    k0, v0 = kc.clone(), vc.clone()
    out = paged_kv_append(k, v, kc, vc, table, lengths, q=q, rot_dim=0)
    assert torch.equal(out, q)
    for n, length in enumerate(lengths.tolist()):
        for t in range(50):
            s = length - 50 + t
            if s >= 0 and 0 <= table[n, s // 32] < kc.shape[0]:
                k0[table[n, s // 32], :, s % 32], v0[table[n, s // 32], :, s % 32] = k[n, t], v[n, t]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


def test_a_cache_that_a_graph_saved():
    """An append marks the caches as changed: a graph that saved one refuses its backward."""
    gen = torch.Generator(DEV).manual_seed(10)
    kc, vc, table = _cache(1, 32, 1, 64, 16, torch.bfloat16, gen)
    w = torch.randn(64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = (kc * w).sum()
    k = torch.randn(1, 1, 1, 64, generator=gen, device=DEV).bfloat16()
    paged_kv_append(k, k, kc, vc, table, torch.tensor([3], device=DEV))
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_captured_serving_steps():
    """An append and two attentions in two graphs on one pool, with other tokens, lengths, pages and bounds at every replay."""
    gen = torch.Generator(DEV).manual_seed(11)
    n, hq, hkv, d = 3, 4, 2, 128
    kc, vc, table = _cache(n, 700, hkv, d, 16, torch.bfloat16, gen)
    start = [c.clone() for c in (kc, vc, table)]
    q, k, v = (torch.randn(1, 9, h, d, generator=gen, device=DEV).bfloat16() for h in (hq, hkv, hkv))
    cu_host = torch.tensor([0, 4, 8, 9])
    cu, lengths = cu_host.to(DEV), torch.tensor([650, 9, 300], device=DEV)
    tree = torch.ones(1, 9, dtype=torch.int64, device=DEV)

    def step(win):
        rows = paged_kv_append(k, v, kc, vc, table, lengths, q=q, rot_dim=64, cu_seqlens=cu, cu_seqlens_cpu=cu_host)
        return [rows] + [paged_attention(rows, kc, vc, table, lengths, window=win, sinks=2, tree=w, cu_seqlens=cu,
                                         cu_seqlens_cpu=cu_host) for w in (None, tree)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(None), step(100)
    torch.cuda.current_stream().wait_stream(s)
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for win in (None, 100):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            outs.append(step(win))
    # as many tokens for each; none for one; tokens before the first sequence and behind the last; lengths on both sides of runs
    for bounds, lens in (([0, 4, 8, 9], [650, 9, 300]), ([0, 4, 4, 9], [1, 0, 700]), ([2, 3, 5, 7], [699, 40, 65]),
                         ([0, 9, 9, 9], [9, 5, 5])):
        fresh = [torch.randn(y.shape, generator=gen, device=DEV).bfloat16() for y in (q, k, v)]
        for y, z in zip((q, k, v), fresh):
            y.copy_(z)
        cu.copy_(torch.tensor(bounds))
        lengths.copy_(torch.tensor(lens))
        tree.copy_(torch.randint(0, 512, (1, 9), generator=gen, device=DEV))
        table.copy_(start[2].flatten()[torch.randperm(table.numel(), generator=gen, device=DEV)].reshape(table.shape))
        for graph, out, win in zip(graphs, outs, (None, 100)):
            kc.copy_(start[0])
            vc.copy_(start[1])
            graph.replay()
            torch.cuda.synchronize()
            rows, plain, drafted = (y.clone() for y in out)
            assert not rows[:, :bounds[0]].any() and not rows[:, bounds[-1]:].any()
            check(plain, reference(rows, kc, vc, table, lengths, win, 2, d**-0.5, None, bounds), "o")
            check(drafted, reference(rows, kc, vc, table, lengths, win, 2, d**-0.5, tree, bounds), "o")
            for m, (a, e) in enumerate(zip(bounds[:-1], bounds[1:])):
                fits = min(e - a, lens[m])
                assert e == a or torch.equal(gather(vc, table[m], lens[m])[lens[m] - fits:], v[0, e - fits:e])


def test_other_streams_and_calls_at_once():
    want = []
    cases = [_case(CASES[i], torch.bfloat16, seed=12) for i in (2, 10, 8)]
    for x in cases:
        want.append(_attend(*x))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(6)]
    got = []
    for j, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append(_attend(*cases[j % 3]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[j % 3]) for j, g in enumerate(got))


def test_views_of_queries_and_no_tokens():
    x = list(_case(CASES[11], torch.bfloat16, seed=13))
    want = _attend(*x)
    q = x[0]
    wide = torch.cat([q, q], 2)[:, :, :q.shape[2]]
    assert not wide.is_contiguous() and torch.equal(_attend(wide, *x[1:]), want)
    head_major = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(_attend(head_major, *x[1:]), want)
    table = torch.cat([x[3], x[3]], 1)[:, :x[3].shape[1]]  # a row stride
    assert torch.equal(_attend(q, x[1], x[2], table, *x[4:]), want)
    columns = x[3].t().contiguous().t()
    assert torch.equal(_attend(q, x[1], x[2], columns, *x[4:]), want)
    assert paged_attention(q[:, :0], *x[1:5]).shape == (2, 0, 4, 128)
    k = torch.zeros(2, 0, 4, 128, device=DEV, dtype=torch.bfloat16)
    before = x[1].clone()
    assert paged_kv_append(k, k, *x[1:5], q=q[:, :0]).shape == (2, 0, 4, 128) and torch.equal(x[1], before)


def test_a_compiled_function_calls_them():
    x = _case(CASES[2], torch.bfloat16, seed=14)
    want = _attend(*x)
    q, kc, vc, table, lengths = x[:5]
    assert torch.equal(torch.compile(lambda y: paged_attention(y * 1.0, kc, vc, table, lengths))(q), want)
