"""64-bit references of attention with a window and sinks, whole sequences and paged caches, with bounds on how far a kernel may
be off that are derived here, term by term.

u = 2^-24, h = half a step of the inputs' type. Scores are sums of D exact products in fp32, off by e_s = scale D u |q|.|k|
(the terms' magnitudes); a weight p by 2 e_s + 2^-21 of itself (the exponential, the row's sum or logarithm, the products with
log2(e)) and, as an operand, by h more. fp16 operands below 2^-14 keep steps of 2^-24 of the row's largest weight: 2^-25 a term,
against a row sum of 1 at least.

  o       Sum p |v| (h + e_p) (+ 2^-25 Sum |v| in fp16)
  dv      Sum p |do| (h + e_p)
  delta   the o that was stored: |do|.(h |o| + its own bound) + D u |do|.|o|
  ds      p (D u |do|.|v| + delta's) + |ds| (h + e_p)
  dq, dk  scale Sum of ds' times |k|, |q|
A sum of n terms in fp32 adds n u of the magnitudes.
"""
from __future__ import annotations

import torch

F64 = torch.float64
U = 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def seen(i, j, window, sinks):
    """[len(i), len(j)]: whether the query at place i sees place j."""
    ok = j[None] <= i[:, None]
    return ok if window is None else ok & ((i[:, None] - j[None] < window) | (j[None] < sinks))


def one_head(q, k, v, mask, scale, h, f16=False, do=None):
    """o [, dq, dk, dv] of one head's rows, each with its bound; q, do [T,D], k, v [L,D], mask [T,L]."""
    q, k, v = q.double(), k.double(), v.double()
    d = q.shape[1]
    s = (q @ k.T) * scale
    e_s = scale * d * U * (q.abs() @ k.abs().T)
    s = torch.where(mask, s, -torch.inf)
    top = s.amax(1, keepdim=True)
    top = torch.where(top.isfinite(), top, 0)
    p = torch.exp(s - top)
    total = p.sum(1, keepdim=True)
    p = torch.where(total > 0, p / total, 0)
    n = k.shape[0] + d
    e_p = 2 * torch.where(mask, e_s, 0).amax(1, keepdim=True) + 2.0**-21 + n * U
    o, mag = p @ v, p @ v.abs()
    o_tol = mag * (h + e_p) + (2.0**-25 * (mask.double() @ v.abs()) if f16 else 0)
    if do is None:
        return o, o_tol
    do = do.double()
    delta = (do * o).sum(1, keepdim=True)
    d_tol = (do.abs() * (h * o.abs() + o_tol)).sum(1, keepdim=True) + d * U * (do.abs() * o.abs()).sum(1, keepdim=True)
    ds = p * (do @ v.T - delta)
    ds_tol = p * (d * U * (do.abs() @ v.abs().T) + d_tol) + ds.abs() * (h + e_p)
    nq = q.shape[0] + d
    more = n * U * ds.abs()
    dq, dq_tol = scale * (ds @ k), scale * ((ds_tol + more) @ k.abs())
    dk, dk_tol = scale * (ds.T @ q), scale * ((ds_tol + nq * U * ds.abs()).T @ q.abs())
    pt = p * (h + e_p + nq * U)
    return o, o_tol, dq, dq_tol, dk, dk_tol, p.T @ do, pt.T @ do.abs()


def window_attention(q, k, v, window, sinks, scale, cu=None, do=None):
    """dict of o and, with ``do``, dq, dk, dv, each with its ``*_tol``."""
    b, t, hq, d = q.shape
    hkv = k.shape[2]
    rep, h = hq // hkv, half_step(q.dtype)
    spans = [(i, 0, t) for i in range(b)] if cu is None else [(0, s, e) for s, e in zip(cu[:-1], cu[1:])]
    names = ("o", "o_tol") + (("dq", "dq_tol", "dk", "dk_tol", "dv", "dv_tol") if do is not None else ())
    out = {m: torch.zeros((k if m[:2] in ("dk", "dv") else q).shape, dtype=F64, device=q.device) for m in names}
    for bi, s, e in spans:
        if s == e:
            continue
        at = torch.arange(e - s, device=q.device)
        mask = seen(at, at, window, sinks)
        for i in range(hq):
            got = one_head(q[bi, s:e, i], k[bi, s:e, i // rep], v[bi, s:e, i // rep], mask, scale, h,
                           q.dtype == torch.float16, None if do is None else do[bi, s:e, i])
            for m, x in zip(names, got):
                if m[:2] in ("dk", "dv"):
                    out[m][bi, s:e, i // rep] += x
                else:
                    out[m][bi, s:e, i] = x
    return out


def gather(cache, table, length):
    """[length, HKV, D] of one sequence's rows; rows on pages that are none hold NaN."""
    pages, hkv, size, d = cache.shape
    out = torch.full((length, hkv, d), torch.nan, dtype=cache.dtype, device=cache.device)
    for s in range(length):
        page = int(table[s // size])
        if 0 <= page < pages:
            out[s] = cache[page, :, s % size]
    return out


def paged_attention(q, kc, vc, table, lengths, window, sinks, scale, tree=None, cu=None):
    """dict of o and o_tol."""
    b, t, hq, d = q.shape
    pages, hkv, size, _ = kc.shape
    rep, h = hq // hkv, half_step(q.dtype)
    spans = [(i, 0, t) for i in range(b)] if cu is None else [(0, s, e) for s, e in zip(cu[:-1], cu[1:])]
    out = {m: torch.zeros(q.shape, dtype=F64, device=q.device) for m in ("o", "o_tol")}
    for n, (bi, s, e) in enumerate(spans):
        length, count = int(lengths[n]), e - s
        if not length:
            continue
        k, v = gather(kc, table[n], length), gather(vc, table[n], length)
        there = (0 <= table[n].long()) & (table[n].long() < pages)
        j = torch.arange(length, device=q.device)
        there = there[j // size]
        base = length - count
        if tree is None:
            mask = seen(base + torch.arange(count, device=q.device), j, window, sinks)
        else:
            words = [int(x) & (1 << count) - 1 for x in tree[bi, s:e]]
            place = torch.tensor([base + bin(x).count("1") - 1 for x in words], device=q.device)
            mask = seen(place, j, window, sinks) & (j < base)
            for r, x in enumerate(words):
                for c in range(count):
                    if x >> c & 1 and base + c >= 0:
                        mask[r, base + c] = True
        mask &= there
        k, v = (torch.where(there[:, None, None], x, 0) for x in (k, v))
        for i in range(hq):
            out["o"][bi, s:e, i], out["o_tol"][bi, s:e, i] = one_head(q[bi, s:e, i], k[:, i // rep], v[:, i // rep], mask,
                                                                      scale, h, q.dtype == torch.float16)
    return out


def check(got, ref, name):
    """|got - ref| <= the bound and one rounding to got's type (and its smallest step)."""
    want, tol = ref[name], ref[name + "_tol"]
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = (got.double() - want).abs()
    step = half_step(got.dtype)
    bound = tol + step * (want.abs() + tol) + torch.finfo(got.dtype).smallest_normal * step
    bad = ~(off <= bound)
    assert not bad.any(), (name, int(bad.sum()), bad.nonzero()[0].tolist(), float((off / bound).nan_to_num(9e9).max()))
