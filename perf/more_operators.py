"""Performance cases of attention with a window and sinks, and of the paged cache of keys and values that serves it.

Every case is one call (or one forward and backward) through the public entry points of ``sorernn_amd``:

- ``window``: ``window_attention``, prompts and training;
- ``append``: ``paged_kv_append``, the new tokens' keys and values normed, rotated and written into their pages, queries beside
  them;
- ``cached``: ``paged_attention``, single tokens, pieces of a prompt and trees of drafted tokens over the pages.

With ``own`` false, ``run`` computes the same results in plain torch (products, sums, exp, comparisons, indexing) in 32 bits.
``exact`` gives them in 64 bits from the formulas.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
THETA = 1e7


def listed():
    return [
        # a short odd prompt of one user, heads of 64: launches count
        {"name": "window_short", "kind": "window", "B": 1, "T": 333, "docs": 0, "HQ": 4, "HKV": 1, "D": 64, "window": 64,
         "sinks": 4, "dtype": "bf16", "train": False},
        # a long prompt of one user
        {"name": "window_prompt", "kind": "window", "B": 1, "T": 8192, "docs": 0, "HQ": 16, "HKV": 4, "D": 128,
         "window": 1024, "sinks": 4, "dtype": "bf16", "train": False},
        # a training step's attention layer
        {"name": "window_train", "kind": "window", "B": 2, "T": 4096, "docs": 0, "HQ": 16, "HKV": 4, "D": 128,
         "window": 1024, "sinks": 4, "dtype": "bf16", "train": True},
        # training on packed documents of uneven lengths, heads of 64, a short window
        {"name": "window_docs_train", "kind": "window", "B": 1, "T": 5003, "docs": 7, "HQ": 8, "HKV": 2, "D": 64,
         "window": 200, "sinks": 1, "dtype": "bf16", "train": True},
        # one token of one sequence: launches and the host's work count
        {"name": "append_1", "kind": "append", "N": 1, "T": 1, "HQ": 16, "HKV": 4, "D": 128, "rot": 32, "norm": True,
         "cached": 1000, "page": 64, "dtype": "bf16"},
        # a serving batch's step
        {"name": "append_64", "kind": "append", "N": 64, "T": 1, "HQ": 16, "HKV": 4, "D": 128, "rot": 32, "norm": True,
         "cached": 500, "page": 16, "dtype": "bf16"},
        # eight prompts enter the cache, whole heads rotated
        {"name": "append_prompts", "kind": "append", "N": 8, "T": 2048, "HQ": 16, "HKV": 4, "D": 128, "rot": 128,
         "norm": False, "cached": 0, "page": 64, "dtype": "fp16"},
        # one token of one sequence with a long cache: the work has to be split over the keys
        {"name": "cached_1", "kind": "cached", "N": 1, "T": 1, "HQ": 16, "HKV": 4, "D": 128, "longest": 32768, "page": 64,
         "window": 0, "sinks": 0, "tree": False, "dtype": "bf16"},
        # a serving batch's step, uneven lengths: a gigabyte of keys and values
        {"name": "cached_64", "kind": "cached", "N": 64, "T": 1, "HQ": 16, "HKV": 4, "D": 128, "longest": 8192, "page": 16,
         "window": 0, "sinks": 0, "tree": False, "dtype": "bf16"},
        # the same with a window and sinks, heads of 64
        {"name": "cached_window", "kind": "cached", "N": 64, "T": 1, "HQ": 16, "HKV": 8, "D": 64, "longest": 8192, "page": 64,
         "window": 1024, "sinks": 4, "tree": False, "dtype": "fp16"},
        # a piece of four prompts over what is cached of them
        {"name": "cached_piece", "kind": "cached", "N": 4, "T": 512, "HQ": 16, "HKV": 4, "D": 128, "longest": 8192,
         "page": 64, "window": 0, "sinks": 0, "tree": False, "dtype": "bf16"},
        # trees of drafted tokens being scored
        {"name": "cached_trees", "kind": "cached", "N": 8, "T": 61, "HQ": 16, "HKV": 4, "D": 128, "longest": 4096, "page": 32,
         "window": 0, "sinks": 0, "tree": True, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["window", "window", "append", "cached", "cached"])
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([r for r in (1, 2, 3, 4, 8, 16) if hkv * r <= 16])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "window":
        train = rng.random() < 0.5
        tokens = _log_int(rng, 1, 4096 if train else 8192)
        docs = rng.choice([0, 0, 1]) and rng.randint(1, max(1, min(20, tokens // 2)))
        b = 1 if docs else rng.choice([x for x in (1, 1, 2, 3) if x <= tokens])
        return {"kind": kind, "B": b, "T": max(1, tokens // b), "docs": docs, "HQ": hq, "HKV": hkv, "D": d,
                "window": rng.choice([0, _log_int(rng, 1, 2048)]), "sinks": rng.choice([0, 1, 4, 33]),
                "dtype": "bf16" if train else dtype, "train": train}
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        n = _log_int(rng, 1, 64)
        return {"kind": kind, "N": n, "T": _log_int(rng, 1, 16384 // n), "HQ": hq, "HKV": hkv, "D": d,
                "rot": rng.choice([0, 16, 32, 64]), "norm": rng.random() < 0.5, "cached": _log_int(rng, 1, 600), "page": page,
                "dtype": dtype}
    n = _log_int(rng, 1, 64)
    longest = _log_int(rng, 64, min(32768, 524288 // n))
    tree = rng.random() < 0.3
    t = _log_int(rng, 1, 64) if tree else rng.choice([1, 1, 2, 5, _log_int(rng, 1, max(1, min(512, 2048 // n)))])
    return {"kind": kind, "N": n, "T": t, "HQ": hq, "HKV": hkv, "D": d, "longest": max(longest, t), "page": page,
            "window": 0 if tree else rng.choice([0, 0, _log_int(rng, 1, 4096)]), "sinks": rng.choice([0, 4]), "tree": tree,
            "dtype": dtype}


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _doc_lens(case):
    """Uneven lengths of the packed documents, one token at least each; a part of the case."""
    total, docs = case["T"], case["docs"]
    if not docs:
        return []
    rng = random.Random(1000 * total + docs)
    share = [rng.random() + 0.1 for _ in range(docs)]
    lens = [1 + int((total - docs) * s / sum(share)) for s in share]
    lens[-1] += total - sum(lens)
    return lens


def _cache_lens(case):
    """Each sequence's tokens in the cache, the new ones counted; a part of the case."""
    n, t = case["N"], case["T"]
    rng = random.Random(n * 7919 + t)
    if case["kind"] == "append":
        return [t + rng.randint(0, case["cached"]) for _ in range(n)]
    longest = case["longest"]
    return [longest] + [rng.randint(max(t, longest // 4), longest) for _ in range(n - 1)]


def _trees(case, seed):
    """[N][T] bits of the drafted tokens that each drafted token sees: itself and its ancestors."""
    rng = random.Random(seed)
    rows = []
    for _ in range(case["N"]):
        bits = []
        for i in range(case["T"]):
            parent = rng.randint(max(-1, i - 9), i - 1)
            bits.append((bits[parent] if parent >= 0 else 0) | 1 << i)
        rows.append(bits)
    return rows


def _raw(case, seed):
    """The case's inputs as a dict of tensors on the GPU, without gradients."""
    gen = torch.Generator(DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hkv, d = case["HQ"], case["HKV"], case["D"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    x = {}
    if case["kind"] == "window":
        b, t = case["B"], case["T"]
        # q and k as a norm leaves them, v as a projection does
        x["q"], x["k"], x["v"] = randn(b, t, hq, d).to(dt), randn(b, t, hkv, d).to(dt), randn(b, t, hkv, d).to(dt)
        lens = _doc_lens(case)
        x["cu_host"] = torch.tensor([0] + lens).cumsum(0) if lens else None
        x["cu"] = x["cu_host"].to(DEV) if lens else None
        if case["train"]:
            x["do"] = randn(b, t, hq, d).to(dt)
        return x
    n, t, page = case["N"], case["T"], case["page"]
    lens = _cache_lens(case)
    width = -(-max(lens) // page)
    x["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    # pages in any order, as a server's free list leaves them
    x["table"] = torch.randperm(n * width, generator=gen, device=DEV).to(torch.int32).reshape(n, width)
    x["kc"] = torch.empty(n * width, hkv, page, d, dtype=dt, device=DEV).normal_(generator=gen)
    x["vc"] = torch.empty(n * width, hkv, page, d, dtype=dt, device=DEV).normal_(generator=gen)
    if case["kind"] == "append":
        # column slices of one fused projection's output, as a layer has them
        proj = (randn(n, t, (hq + 2 * hkv) * d) * 0.7).to(dt)
        x["q"], x["k"], x["v"] = (y.unflatten(-1, (-1, d)) for y in proj.split([hq * d, hkv * d, hkv * d], -1))
        x["qw"], x["kw"] = (1 + 0.1 * randn(d), 1 + 0.1 * randn(d)) if case["norm"] else (None, None)
        return x
    x["q"] = randn(n, t, hq, d).to(dt)
    x["tree"] = None
    if case["tree"]:
        bits = [[b - (1 << 64) if b >> 63 else b for b in row] for row in _trees(case, seed)]
        x["tree"] = torch.tensor(bits, dtype=torch.int64, device=DEV)
    return x


def prepare(case, seed):
    x = _raw(case, seed)
    leaves = []
    if case.get("train"):
        leaves = ["q", "k", "v"]
        for name in leaves:
            x[name].requires_grad_(True)
    return {"case": case, "x": x, "leaves": leaves}


# ---------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------
def _plain_softmax_product(q, k, v, mask):
    """softmax of the visible scores times v: ``q [N,HKV,R,D]``, ``k, v [N,HKV,L,D]``, ``mask [N,1,R,L]``; 0 where a row sees
    nothing."""
    s = (q @ k.transpose(-1, -2).contiguous()) * q.shape[-1] ** -0.5
    s = s.masked_fill(~mask, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(torch.finfo(s.dtype).min).detach()
    p = (s - top).exp()
    return (p @ v) / p.sum(-1, keepdim=True).clamp_min(torch.finfo(s.dtype).tiny)


def _plain_window(q, k, v, window, sinks, cu):
    b, t, hq, d = q.shape
    hkv = k.shape[2]
    place = torch.arange(t, device=DEV)
    doc = torch.zeros_like(place)
    if cu is not None:
        doc = torch.searchsorted(cu, place, right=True) - 1
        place = place - cu[doc]
    i, j = place[:, None], place[None, :]
    mask = (doc[:, None] == doc[None, :]) & (j <= i)
    if window:
        mask &= (i - j < window) | (j < sinks)
    rows = q.float().reshape(b, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    o = _plain_softmax_product(rows, k.float().transpose(1, 2).contiguous(), v.float().transpose(1, 2).contiguous(),
                               mask.repeat(hq // hkv, 1)[None, None])
    return o.reshape(b, hq, t, d).transpose(1, 2).to(q.dtype)


def _plain_rows(x, w, pos, rot):
    """RMSNorm of the last axis (with ``w``), then the rotation of its first ``rot`` entries; angles in 64 bits."""
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w
    half = rot // 2
    inv = THETA ** (-torch.arange(half, device=x.device, dtype=torch.float64) / max(half, 1))
    angle = (pos.double()[..., None] * inv)[:, :, None, :]
    cos, sin = angle.cos().float(), angle.sin().float()
    lo, hi = y[..., :half], y[..., half:rot]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, y[..., rot:]], -1).to(x.dtype)


def _plain_append(case, x):
    pos = x["lengths"].long()[:, None] - case["T"] + torch.arange(case["T"], device=DEV)
    page = x["table"].long().gather(1, pos // case["page"])
    q = _plain_rows(x["q"], x["qw"], pos, case["rot"])
    x["kc"][page, :, pos % case["page"]] = _plain_rows(x["k"], x["kw"], pos, case["rot"])
    x["vc"][page, :, pos % case["page"]] = x["v"]
    return [q, x["kc"], x["vc"]]


def _plain_cached(case, x):
    n, t, hq, hkv, d = (case[m] for m in ("N", "T", "HQ", "HKV", "D"))
    longest = x["table"].shape[1] * case["page"]
    rep = hq // hkv
    k, v = (c[x["table"].long()].transpose(1, 2).reshape(n, hkv, longest, d).float() for c in (x["kc"], x["vc"]))
    first = (x["lengths"].long() - t)[:, None, None]
    i, j = first + torch.arange(t, device=DEV)[:, None], torch.arange(longest, device=DEV)
    mask = j <= i
    if case["window"]:
        mask &= (i - j < case["window"]) | (j < case["sinks"])
    if x["tree"] is not None:
        mask = (j < first) | ((j < first + t) & ((x["tree"][..., None] >> (j - first).clamp(0, 63)) & 1).bool())
    rows = x["q"].float().reshape(n, t, hkv, rep, d).transpose(1, 2).reshape(n, hkv, t * rep, d)
    o = _plain_softmax_product(rows, k, v, mask.repeat_interleave(rep, 1)[:, None])
    return o.reshape(n, hkv, t, rep, d).transpose(1, 2).reshape(n, t, hq, d).to(x["q"].dtype)


def run(state):
    case, x = state["case"], state["x"]
    if case["kind"] == "append":
        if not own:
            return _plain_append(case, x)
        from sorernn_amd import paged_kv_append

        q = paged_kv_append(x["k"], x["v"], x["kc"], x["vc"], x["table"], x["lengths"], q=x["q"], q_weight=x["qw"],
                            k_weight=x["kw"], rot_dim=case["rot"], theta=THETA, eps=EPS)
        return [q, x["kc"], x["vc"]]
    if case["kind"] == "cached":
        if not own:
            return _plain_cached(case, x)
        from sorernn_amd import paged_attention

        return paged_attention(x["q"], x["kc"], x["vc"], x["table"], x["lengths"], window=case["window"] or None,
                               sinks=case["sinks"], tree=x["tree"])
    if own:
        from sorernn_amd import window_attention

        o = window_attention(x["q"], x["k"], x["v"], window=case["window"] or None, sinks=case["sinks"],
                             cu_seqlens=x["cu"], cu_seqlens_cpu=x["cu_host"])
    else:
        o = _plain_window(x["q"], x["k"], x["v"], case["window"], case["sinks"], x["cu"])
    if not case["train"]:
        return o
    return [o.detach(), *torch.autograd.grad([o], [x[m] for m in state["leaves"]], [x["do"]])]


# ---------------------------------------------------------------------------------------------------
# the formulas in 64 bits
# ---------------------------------------------------------------------------------------------------
def _weights(q, k, seen):
    """Softmax of one head's visible scores, ``q [T,D]``, ``k [L,D]``."""
    s = torch.where(seen, q @ k.T * q.shape[1] ** -0.5, -math.inf)
    e = torch.exp(s - s.max(1, keepdim=True).values)
    return e / e.sum(1, keepdim=True)


def _seen(i, j, window, sinks):
    seen = i[:, None] >= j[None]
    return seen & ((i[:, None] - j[None] < window) | (j[None] < sinks)) if window else seen


def _exact_window(case, x):
    b, t, hq, hkv, d = (case[m] for m in ("B", "T", "HQ", "HKV", "D"))
    rep, scale = hq // hkv, d**-0.5
    q, k, v = (x[m].detach().double() for m in ("q", "k", "v"))
    lens = _doc_lens(case)
    spans = [(0, sum(lens[:i]), sum(lens[:i + 1])) for i in range(len(lens))] if lens else [(i, 0, t) for i in range(b)]
    o = torch.empty_like(q)
    dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for bi, s, e in spans:
        place = torch.arange(e - s, device=DEV)
        seen = _seen(place, place, case["window"], case["sinks"])
        for h in range(hq):
            qh, kh, vh = q[bi, s:e, h], k[bi, s:e, h // rep], v[bi, s:e, h // rep]
            p = _weights(qh, kh, seen)
            oh = o[bi, s:e, h] = p @ vh
            if case["train"]:
                up = x["do"][bi, s:e, h].double()
                ds = p * (up @ vh.T - (up * oh).sum(1, keepdim=True)) * scale
                dq[bi, s:e, h] = ds @ kh
                dk[bi, s:e, h // rep] += ds.T @ qh
                dv[bi, s:e, h // rep] += p.T @ up
    return [o, dq, dk, dv] if case["train"] else o


def _exact_rows(x, w, pos, rot):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + EPS) * w.double()
    if not rot:
        return y
    freq = torch.tensor([THETA ** (-2.0 * f / rot) for f in range(rot // 2)], dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.ones(*pos.shape, 1, rot // 2, dtype=torch.float64, device=DEV), pos.double()[..., None, None] * freq)
    c = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * turn
    return torch.cat([c.real, c.imag, y[..., rot:]], -1)


def _exact_append(case, x):
    t, page = case["T"], case["page"]
    lens = _cache_lens(case)
    pos = torch.tensor([[m - t + i for i in range(t)] for m in lens], device=DEV)
    kc, vc = x["kc"].double(), x["vc"].double()
    k = _exact_rows(x["k"], x["kw"], pos, case["rot"])
    for n, row in enumerate(x["table"].tolist()):
        slots = torch.tensor([row[p // page] * page + p % page for p in range(lens[n] - t, lens[n])], device=DEV)
        for h in range(case["HKV"]):
            for cache, new in ((kc, k), (vc, x["v"].double())):
                cache.transpose(0, 1)[h][slots // page, slots % page] = new[n, :, h]
    return [_exact_rows(x["q"], x["qw"], pos, case["rot"]), kc, vc]


def _exact_cached(case, x, seed):
    n, t, hq, hkv, d, page = (case[m] for m in ("N", "T", "HQ", "HKV", "D", "page"))
    o = torch.empty(n, t, hq, d, dtype=torch.float64, device=DEV)
    trees = _trees(case, seed) if case["tree"] else None
    for m, length in enumerate(_cache_lens(case)):
        pages = x["table"][m, :-(-length // page)].long()
        place = torch.arange(length, device=DEV)
        seen = _seen(place[length - t:], place, case["window"], case["sinks"])
        if trees:
            drafted = [[bool(bits >> i & 1) for i in range(t)] for bits in trees[m]]
            seen = torch.cat([torch.ones(t, length - t, dtype=torch.bool), torch.tensor(drafted)], 1).to(DEV)
        for g in range(hkv):
            k, v = (c[pages, g].reshape(-1, d)[:length].double() for c in (x["kc"], x["vc"]))
            for h in range(g * (hq // hkv), (g + 1) * (hq // hkv)):
                o[m, :, h] = _weights(x["q"][m, :, h].double(), k, seen) @ v
    return o


def exact(case, seed):
    x = _raw(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, x)
    return _exact_window(case, x) if case["kind"] == "window" else _exact_cached(case, x, seed)


def _pairs(first, last, window, sinks):
    """Visible pairs of the queries at places ``first .. last - 1`` of one sequence."""
    return sum(i + 1 if not window or i < window else window + min(sinks, i + 1 - window) for i in range(first, last))


def work(case):
    hq, hkv, d = case["HQ"], case["HKV"], case["D"]
    if case["kind"] == "append":
        tokens = case["N"] * case["T"]
        rows = tokens * (hq + 2 * hkv) * d * 2
        return {"bytes": 2 * rows + (8 * d if case["norm"] else 0) + 4 * tokens, "flops": tokens * (hq + hkv) * d * 8}
    window, sinks = case["window"], case["sinks"]
    if case["kind"] == "window":
        lens = _doc_lens(case) or [case["T"]] * case["B"]
        pairs = sum(_pairs(0, n, window, sinks) for n in lens)
        total = sum(lens) * d * 2
        size = total * (2 * hq + 2 * hkv)
        if case["train"]:  # besides: q, k, v, o, do read, dq, dk, dv written
            size += total * (4 * hq + 4 * hkv)
        return {"bytes": size, "flops": pairs * hq * d * (14 if case["train"] else 4)}
    t = case["T"]
    pairs = seen = 0
    for m, length in enumerate(_cache_lens(case)):
        if case["tree"]:  # about six ancestors
            pairs += t * (length - t + 6)
        else:
            pairs += _pairs(length - t, length, window, sinks)
        seen += min(length, window + t - 1 + sinks) if window else length
    return {"bytes": (2 * case["N"] * t * hq + 2 * seen * hkv) * d * 2, "flops": 4 * pairs * hq * d}
