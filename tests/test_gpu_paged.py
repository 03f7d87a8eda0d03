"""GPU: the paged cache of keys and values: appending with norm and rotation, and attention over it, against 64 bits.

Bounds of the attention: tests/window_ref.py. Appended rows are computed in fp32: products and a root (4 u), a sum of D squares
(D u / 2 of the factor), the angle's rounding to fp32 (2^-22 of a turn's values) and two products: (D + 24) u of the terms'
magnitudes, then one rounding; values are copied.
"""
import pytest
import torch

from sorernn_amd import paged_attention, paged_kv_append
from tests.linear_ref import check as check_rows, norm_rope
from tests.window_ref import check, gather, paged_attention as reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24


def _cache(n, longest, hkv, d, page, dtype, gen, layout="heads", spare=3):
    """Caches with pages in any order and a table: [pages, HKV, page, D], or tokens before heads and a view of it."""
    width = -(-longest // page)
    pages = n * width + spare
    shape = (pages, hkv, page, d) if layout == "heads" else (pages, page, hkv, d)
    kc, vc = (torch.randn(shape, generator=gen, device=DEV).to(dtype) for _ in range(2))
    if layout != "heads":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    table = torch.randperm(pages, generator=gen, device=DEV)[:n * width].to(torch.int32).reshape(n, width)
    return kc, vc, table


def _tree(n, t, gen):
    """[N,T] words: itself and its ancestors, each token below one of the few before it."""
    words = torch.zeros(n, t, dtype=torch.int64)
    for i in range(n):
        for j in range(t):
            parent = int(torch.randint(max(-1, j - 5), j, (1,), generator=gen)) if j else -1
            bits = (int(words[i, parent]) if parent >= 0 else 0) & (1 << 64) - 1 | 1 << j
            words[i, j] = bits - (1 << 64) if bits >> 63 else bits
    return words


CASES = [
    # lengths, T (or new tokens a sequence), HQ, HKV, D, page, window, sinks, tree, layout
    ([1], 1, 1, 1, 64, 16, None, 0, False, "heads"),
    ([17, 1, 16, 33], 1, 4, 2, 128, 16, None, 0, False, "heads"),
    ([500, 1000, 3], 1, 16, 4, 128, 64, None, 0, False, "tokens"),
    ([700, 90], 1, 40, 1, 64, 32, None, 0, False, "heads"),
    ([2000, 31, 0], 1, 3, 1, 128, 128, 100, 3, False, "heads"),
    ([3000, 640], 2, 8, 8, 64, 64, 64, 0, False, "tokens"),
    ([300, 5, 70], 5, 6, 2, 128, 16, 33, 40, False, "heads"),
    ([900, 61], 61, 4, 1, 128, 32, None, 0, True, "heads"),
    ([700, 64, 130], 64, 2, 2, 64, 16, 50, 4, True, "tokens"),
    ([40, 1], 1, 2, 1, 64, 16, None, 0, True, "heads"),
    ([400, 129, 1000], 129, 8, 2, 64, 16, None, 0, False, "heads"),
    ([1500, 300], 300, 4, 4, 128, 64, 200, 5, False, "tokens"),
    ([333, 333], 333, 4, 1, 128, 32, None, 0, False, "heads"),
    ([500, 40, 3, 900, 77], [1, 40, 2, 7, 1], 4, 1, 128, 16, None, 0, False, "heads"),
    ([500, 40, 64, 900], [1, 40, 64, 7], 4, 2, 64, 32, 60, 2, True, "heads"),
    ([900, 600, 1], [700, 600, 1], 2, 1, 64, 64, 128, 1, False, "tokens"),
    # padded in front: fewer tokens than rows; rows at places below 0 see nothing
    ([5, 100, 0], 20, 4, 2, 128, 16, None, 0, False, "heads"),
    ([5, 300, 129], 140, 8, 4, 64, 16, 17, 2, False, "heads"),
]
IDS = [f"l{'.'.join(map(str, c[0]))}-t{c[1] if isinstance(c[1], int) else '.'.join(map(str, c[1]))}-h{c[2]}.{c[3]}-{c[4]}-p{c[5]}"
       f"-w{c[6]}.{c[7]}{'-tree' if c[8] else ''}-{c[9]}" for c in CASES]


def _case(case, dtype, seed=0):
    lengths, t, hq, hkv, d, page, win, sinks, tree, layout = case
    gen = torch.Generator(DEV).manual_seed(seed)
    n = len(lengths)
    kc, vc, table = _cache(n, max(max(lengths), 1), hkv, d, page, dtype, gen, layout)
    uneven = not isinstance(t, int)
    bounds = [0] + torch.tensor(t).cumsum(0).tolist() if uneven else None
    q = torch.randn(*((1, sum(t)) if uneven else (n, t)), hq, d, generator=gen, device=DEV).to(dtype)
    words = None
    if tree:
        host = torch.Generator().manual_seed(seed)
        words = torch.cat([_tree(1, m, host) for m in t], 1) if uneven else _tree(n, t, host)
        words = words.to(DEV)
    return q, kc, vc, table, torch.tensor(lengths, device=DEV), win, sinks, words, bounds


def _attend(q, kc, vc, table, lengths, win, sinks, words, bounds, **kw):
    cu = None if bounds is None else torch.tensor(bounds)
    return paged_attention(q, kc, vc, table, lengths, window=win, sinks=sinks, tree=words, cu_seqlens=None if cu is None else cu.to(DEV),
                           cu_seqlens_cpu=cu, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_attention(case, dtype):
    x = _case(case, dtype)
    o = _attend(*x)
    assert o.dtype == dtype and o.is_contiguous()
    q, kc, vc, table, lengths, win, sinks, words, bounds = x
    check(o, reference(q, kc, vc, table, lengths, win, sinks, q.shape[-1] ** -0.5, words, bounds), "o")
    assert torch.equal(o, _attend(q, kc, vc, table, lengths.int(), win, sinks, words, bounds))


APPENDS = [
    # lengths, T, HQ, HKV, D, page, rot, norm, positions, layout
    ([1], 1, 1, 1, 64, 16, 64, True, False, "heads"),
    ([17, 40, 16, 0], 1, 16, 4, 128, 16, 32, True, False, "heads"),
    ([500, 1000, 3], 3, 4, 2, 128, 64, 128, False, True, "tokens"),
    ([300, 301], 300, 5, 5, 64, 32, 16, True, False, "heads"),
    ([60, 5, 300], 70, 0, 3, 128, 16, 48, False, False, "heads"),
    ([60, 5, 300], 70, 2, 1, 64, 16, 0, True, False, "heads"),
    ([500, 40, 3, 900, 77], [1, 40, 2, 7, 1], 4, 1, 128, 16, 64, True, True, "tokens"),
    ([400, 700], [333, 699], 4, 4, 64, 64, 32, False, False, "heads"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"l{'.'.join(map(str, c[0]))}-h{c[2]}.{c[3]}-{c[4]}-p{c[5]}-r{c[6]}")
def test_append(case, dtype):
    lengths, t, hq, hkv, d, page, rot, norm, given, layout = case
    gen = torch.Generator(DEV).manual_seed(3)
    n = len(lengths)
    kc, vc, table = _cache(n, max(lengths), hkv, d, page, dtype, gen, layout)
    k0, v0 = kc.clone(), vc.clone()
    uneven = not isinstance(t, int)
    counts = t if uneven else [t] * n
    b, total = (1, sum(t)) if uneven else (n, t)
    proj = torch.randn(b, total, (hq + 2 * hkv) * d, generator=gen, device=DEV).to(dtype)
    q, k, v = (y.unflatten(-1, (-1, d)) if y.shape[-1] else None for y in proj.split([hq * d, hkv * d, hkv * d], -1))
    qw, kw = ((1 + 0.1 * torch.randn(d, generator=gen, device=DEV)) if norm else None for _ in range(2))
    place = torch.cat([torch.arange(m - c, m) for m, c in zip(lengths, counts)]).reshape(b, total).to(DEV)
    pos = torch.randint(0, 1000000, (b, total), generator=gen, device=DEV) if given else None
    cu = torch.tensor([0] + torch.tensor(t).cumsum(0).tolist()) if uneven else None
    out = paged_kv_append(k, v, kc, vc, table, torch.tensor(lengths, device=DEV), q=q, q_weight=qw if q is not None else None,
                          k_weight=kw, positions=pos, rot_dim=rot, cu_seqlens=None if cu is None else cu.to(DEV),
                          cu_seqlens_cpu=cu)
    at = place if pos is None else pos

    def rows(x, w):
        if w is None:  # a norm that leaves a row as it is: unit mean square
            ref = _rotated(x, at, rot)
        else:
            ref = norm_rope(x, w, at, rot, 1e7, 1e-6) if rot else _normed(x, w)
        return ref

    per = (d + 24) * U
    if q is None:
        assert out is None
    else:
        assert out.is_contiguous() and out.dtype == dtype
        check_rows(out, rows(q, qw), "y", per)
    ref = rows(k, kw)
    flat_k, flat_v = torch.empty_like(k), v
    i = 0
    left_k, left_v = k0.clone(), v0.clone()  # what was there, with the new rows put in
    keep = torch.zeros(b, total, dtype=torch.bool, device=DEV)
    for s in range(n):
        for c in range(counts[s]):
            bi, ti = (0, i) if uneven else (s, c)
            i += 1
            p = lengths[s] - counts[s] + c
            if p < 0:
                continue
            page_no = int(table[s, p // page])
            flat_k[bi, ti] = kc[page_no, :, p % page]
            left_k[page_no, :, p % page] = flat_k[bi, ti]
            left_v[page_no, :, p % page] = flat_v[bi, ti]
            keep[bi, ti] = True
    ref = {m: y[keep][None] for m, y in ref.items() if m in ("y", "y_mag")}
    check_rows(flat_k[keep][None], ref, "y", per)
    assert torch.equal(kc, left_k) and torch.equal(vc, left_v)


def _rotated(x, pos, rot):
    ones = torch.ones(x.shape[-1], device=DEV)
    x = x.double()
    size = (x * x).mean(-1, keepdim=True).sqrt()
    if not rot:
        return {"y": x, "y_mag": x.abs()}
    ref = norm_rope(x / size, ones, pos, rot, 1e7, 0.0)
    return {"y": ref["y"] * size, "y_mag": ref["y_mag"] * size}


def _normed(x, w):
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
    return {"y": y, "y_mag": y.abs()}


def test_a_prompt_in_pieces_then_single_tokens():
    """Appends and attention as a server makes them, and what the whole sequence gives at once. Both round the rotated rows
    once from fp32, but sum a product pair in either order, so they are compared with 64 bits and not with one another."""
    from sorernn_amd import qk_norm_rope, window_attention
    from tests.window_ref import window_attention as whole_reference

    gen = torch.Generator(DEV).manual_seed(5)
    total, hq, hkv, d, win, sinks = 700, 4, 2, 128, 150, 3
    q, k, v = (torch.randn(1, total, h, d, generator=gen, device=DEV).bfloat16() for h in (hq, hkv, hkv))
    qw, kw = (1 + 0.1 * torch.randn(d, generator=gen, device=DEV) for _ in range(2))
    qr, kr = qk_norm_rope(q, k, qw, kw, rot_dim=32)
    whole = window_attention(qr, kr, v, window=win, sinks=sinks)
    kc, vc, table = _cache(1, total, hkv, d, 16, torch.bfloat16, gen)
    at, rows, pieces = 0, [], []
    for t in (300, 1, 257, 5) + (1,) * 137:
        part = slice(at, at + t)
        at += t
        lengths = torch.tensor([at], device=DEV)
        rows.append(paged_kv_append(k[:, part], v[:, part], kc, vc, table, lengths, q=q[:, part], q_weight=qw, k_weight=kw,
                                    rot_dim=32))
        pieces.append(paged_attention(rows[-1], kc, vc, table, lengths, window=win, sinks=sinks))
    assert at == total and torch.equal(gather(vc, table[0], total), v[0])
    place = torch.arange(total, device=DEV)[None]
    cached = gather(kc, table[0], total)[None]
    rows = torch.cat(rows, 1)
    check_rows(rows, norm_rope(q, qw, place, 32, 1e7, 1e-6), "y", (d + 24) * U)
    check_rows(cached, norm_rope(k, kw, place, 32, 1e7, 1e-6), "y", (d + 24) * U)
    check(torch.cat(pieces, 1), reference(rows, kc, vc, table, torch.tensor([total]), win, sinks, d**-0.5), "o")
    check(whole, whole_reference(qr, kr, v, win, sinks, d**-0.5), "o")
