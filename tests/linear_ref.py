"""64-bit references of the decay linear attention operators and of the q/k norm with rotation, token by token, with the
magnitudes that error bounds are made of.

Every result is a sum of products. ``*_mag`` is the same sum over the magnitudes of its terms: if each term has a relative
error of at most d, the result is off by at most d times it, whatever cancels.
"""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def half_step(dtype):
    """The largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def spans(b, t, cu):
    if cu is None:
        return [(i, 0, t) for i in range(b)]
    cu = cu.tolist()
    return [(0, p, e) for p, e in zip(cu[:-1], cu[1:])]


def _rows(x, sp, longest, hv):
    """[B,T,H,W] -> [longest, N, HV, W] in 64 bits, zeros behind each sequence's end."""
    out = torch.zeros(longest, len(sp), hv, x.shape[-1], dtype=F64, device=x.device)
    for i, (bi, p, e) in enumerate(sp):
        out[:e - p, i] = x[bi, p:e].double().repeat_interleave(hv // x.shape[2], 1)
    return out


def _back(y, sp, b, t, heads):
    out = torch.zeros(b, t, heads, y.shape[-1], dtype=F64, device=y.device)
    for i, (bi, p, e) in enumerate(sp):
        out[bi, p:e] = y[:e - p, i].reshape(e - p, heads, y.shape[2] // heads, -1).sum(2)
    return out


def decay_attention(q, k, v, g, scale, h0=None, cu=None, do=None, dht=None):
    """dict of o, state and, with ``do`` (and ``dht``), dq, dk, dv, dg, dh0, each with its ``*_mag``."""
    b, t, h, kd = q.shape
    hv, vd = v.shape[2], v.shape[3]
    sp = spans(b, t, cu)
    n, longest = len(sp), max(e - p for _, p, e in sp)
    g = torch.zeros(b, t, hv, device=q.device) if g is None else (g.expand(b, t, hv) if g.dim() == 1 else g)
    Q, K, V = (_rows(x, sp, longest, hv) for x in (q, k, v))
    a = _rows(g[..., None], sp, longest, hv)[..., 0].exp()[..., None, None]
    zero = torch.zeros(n, hv, kd, vd, dtype=F64, device=q.device)
    S = zero + (h0.double() if h0 is not None else 0)
    M = S.abs()
    o, om = torch.empty_like(V), torch.empty_like(V)
    if do is not None:
        D = _rows(do, sp, longest, hv)
        dq, dqm = torch.empty_like(Q), torch.empty_like(Q)
    for i in range(longest):
        kv = K[i, :, :, :, None] * V[i, :, :, None, :]
        S, M = a[i] * S + kv, a[i] * M + kv.abs()
        o[i] = scale * (Q[i][..., None] * S).sum(2)
        om[i] = abs(scale) * (Q[i].abs()[..., None] * M).sum(2)
        if do is not None:
            dq[i] = scale * (S * D[i][:, :, None]).sum(3)
            dqm[i] = abs(scale) * (M * D[i].abs()[:, :, None]).sum(3)
    r = {"o": _back(o, sp, b, t, hv), "o_mag": _back(om, sp, b, t, hv), "state": S, "state_mag": M}
    if do is None:
        return r
    R = zero + (dht.double() if dht is not None else 0)
    RM, dS = R.abs(), R.clone()
    dk, dkm, dv, dvm = torch.empty_like(Q), torch.empty_like(Q), torch.empty_like(V), torch.empty_like(V)
    for i in reversed(range(longest)):
        step = a[i + 1] if i + 1 < longest else 1.0
        qd = scale * Q[i, :, :, :, None] * D[i, :, :, None, :]
        R, RM = step * R + qd, step * RM + qd.abs()
        dk[i], dkm[i] = (R * V[i][:, :, None]).sum(3), (RM * V[i].abs()[:, :, None]).sum(3)
        dv[i], dvm[i] = (R * K[i][..., None]).sum(2), (RM * K[i].abs()[..., None]).sum(2)
    for nm, x, m, heads in (("dq", dq, dqm, h), ("dk", dk, dkm, h), ("dv", dv, dvm, hv)):
        r[nm], r[nm + "_mag"] = _back(x, sp, b, t, heads), _back(m, sp, b, t, heads)
    each, mag = (Q * dq).sum(3) - (K * dk).sum(3), (Q.abs() * dqm).sum(3) + (K.abs() * dkm).sum(3)
    dg = each.flip(0).cumsum(0).flip(0) + (S * dS).sum((2, 3))
    dgm = mag.flip(0).cumsum(0).flip(0) + (M * dS.abs()).sum((2, 3))
    r["dg"], r["dg_mag"] = (_back(x[..., None], sp, b, t, hv)[..., 0] for x in (dg, dgm))
    r["dh0"], r["dh0_mag"] = a[0] * R, a[0] * RM
    return r


def norm_rope(x, w, pos, rot, theta, eps, up=None):
    """y of one of q, k [B,T,H,D] at positions [B,T] and, with ``up``, dx and dw, each with its ``*_mag``."""
    d, half = x.shape[3], rot // 2
    x = x.double()
    w = torch.ones(d, dtype=F64, device=x.device) if w is None else w.double()
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    freq = torch.tensor([theta ** (-2.0 * f / rot) for f in range(half)], dtype=F64, device=x.device)
    ang = (pos.double()[..., None] * freq)[:, :, None]

    def rotate(y, sign):
        lo, hi = y[..., :half], y[..., half:rot]
        s = sign * ang.sin()
        mag = y.abs().clone()
        mag[..., :half] = mag[..., half:rot] = lo.abs() + hi.abs()
        return torch.cat([lo * ang.cos() - hi * s, hi * ang.cos() + lo * s, y[..., rot:]], -1), mag

    y, mag = rotate(x * r * w, 1)
    out = {"y": y, "y_mag": mag}
    if up is not None:
        dy, dym = rotate(up.double(), -1)
        dn, dnm = dy * w, dym * w.abs()
        out["dx"] = r * dn - x * r**3 * (dn * x).mean(-1, keepdim=True)
        out["dx_mag"] = r * dnm + x.abs() * r**3 * (dnm * x.abs()).mean(-1, keepdim=True)
        out["dw"], out["dw_mag"] = (dy * x * r).sum((0, 1, 2)), (dym * (x * r).abs()).sum((0, 1, 2))
    return out


def check(got, ref, name, per_term):
    """|got - ref| <= one rounding to got's type + per_term times the magnitude of the terms (+ the smallest step)."""
    want, mag = ref[name], ref[name + "_mag"]
    assert got.shape == want.shape, (name, got.shape, want.shape)
    step = half_step(got.dtype)
    err = (got.double() - want).abs()
    bound = step * want.abs() * (1 + 2 * step) + per_term * mag * (1 + step) + torch.finfo(got.dtype).smallest_normal * step * 2
    over = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert math.isfinite(over) and over <= 1.0, f"{name}: {over:.3f} of the bound, largest error {err.max().item():.3e}"
