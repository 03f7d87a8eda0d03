"""Performance cases of the decay linear attention operators and of the q/k norm with rotation before them.

Every case is one call (or one forward and backward) through the public entry points of ``sorernn_amd``:

- ``chunk``: ``chunk_decay_linear_attention``, prompts and training;
- ``recurrent``: ``fused_recurrent_decay_linear_attention``, single tokens and a few tokens from stored states;
- ``rope``: ``qk_norm_rope``, the RMSNorm of every q/k head with the rotation in the same pass.

With ``own`` false, ``run`` computes the same results in plain torch (products, sums, exp, indexing) in 32 bits.
``exact`` gives them in 64 bits from the token-by-token definition.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
CHUNK = 64
EPS = 1e-6
THETA = 1e7


def listed():
    return [
        # one token for one sequence: launches and the host's work count
        {"name": "decode_1", "kind": "recurrent", "B": 1, "T": 1, "H": 16, "HV": 16, "K": 128, "V": 128, "gate": "token",
         "dtype": "bf16", "h0": True},
        # a serving batch: one token for each of 64 sequences, 67 MB of fp32 states read and as many written
        {"name": "decode_64", "kind": "recurrent", "B": 64, "T": 1, "H": 16, "HV": 16, "K": 128, "V": 128, "gate": "head",
         "dtype": "bf16", "h0": True},
        # a few tokens a sequence in full precision, shared q/k heads (a draft being scored, a unit-sized run)
        {"name": "draft_fp32", "kind": "recurrent", "B": 8, "T": 5, "H": 4, "HV": 8, "K": 64, "V": 64, "gate": "token",
         "dtype": "fp32", "h0": True},
        # a short odd prompt of one user, heads of 64, one decay a head
        {"name": "prompt_333", "kind": "chunk", "B": 1, "T": 333, "docs": 0, "H": 4, "HV": 4, "K": 64, "V": 64,
         "gate": "head", "dtype": "bf16", "h0": False, "train": False},
        # the batch prefill of the 0.8B shape, from and to a state
        {"name": "prompt_batch", "kind": "chunk", "B": 4, "T": 4096, "docs": 0, "H": 16, "HV": 16, "K": 128, "V": 128,
         "gate": "token", "dtype": "bf16", "h0": True, "train": False},
        # packed documents of uneven lengths
        {"name": "prompt_docs", "kind": "chunk", "B": 1, "T": 32768, "docs": 8, "H": 16, "HV": 16, "K": 128, "V": 128,
         "gate": "token", "dtype": "bf16", "h0": True, "train": False},
        # one long prompt, where the work has to be split along the sequence
        {"name": "prompt_long", "kind": "chunk", "B": 1, "T": 16384, "docs": 0, "H": 16, "HV": 16, "K": 128, "V": 128,
         "gate": "head", "dtype": "bf16", "h0": False, "train": False},
        # a training step of the operator at the batch prefill's sizes
        {"name": "train_batch", "kind": "chunk", "B": 4, "T": 4096, "docs": 0, "H": 16, "HV": 16, "K": 128, "V": 128,
         "gate": "token", "dtype": "bf16", "h0": False, "train": True},
        # a training step on packed documents of odd lengths, shared q/k heads, different head sizes, states with gradients
        {"name": "train_docs", "kind": "chunk", "B": 1, "T": 3001, "docs": 7, "H": 2, "HV": 4, "K": 64, "V": 128,
         "gate": "token", "dtype": "bf16", "h0": True, "train": True},
        # the norm and rotation of a decode step's rows, far into long texts
        {"name": "rope_decode", "kind": "rope", "B": 64, "T": 1, "HQ": 16, "HK": 16, "D": 128, "rot": 32, "pos": 1000000,
         "dtype": "bf16", "train": False},
        # of a batch prefill's rows, shared keys
        {"name": "rope_batch", "kind": "rope", "B": 4, "T": 4096, "HQ": 16, "HK": 4, "D": 128, "rot": 128, "pos": 0,
         "dtype": "bf16", "train": False},
        # of a training step's rows, with its backward and the weights' gradients
        {"name": "rope_train", "kind": "rope", "B": 4, "T": 4096, "HQ": 16, "HK": 16, "D": 128, "rot": 32, "pos": 0,
         "dtype": "bf16", "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["recurrent", "chunk", "chunk", "chunk", "rope"])
    if kind == "rope":
        d = rng.choice([64, 128, 256])
        hq = rng.choice([1, 2, 3, 4, 8, 16])
        hk = rng.choice([h for h in (1, 2, 3, 4, 8, 16) if hq % h == 0])
        tokens = _log_int(rng, 1, 16384 * 16 * 128 // (16 * d))
        b = rng.choice([x for x in (1, 2, 4, 64) if x <= tokens])
        return {"kind": kind, "B": b, "T": max(1, tokens // b), "HQ": hq, "HK": hk, "D": d,
                "rot": rng.choice([x for x in (16, 32, 64, 128, 256) if x <= d]), "pos": rng.choice([0, 1000, 1000000]),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "train": rng.random() < 0.5}
    rep = rng.choice([1, 1, 1, 2, 4])
    h = rng.choice([1, 2, 4, 8, 16])
    h = max(1, min(h, 16 // rep))
    kd, vd = rng.choice([(64, 64), (128, 128), (64, 128), (128, 64)])
    gate = rng.choice(["token", "token", "head", "none"])
    h0 = rng.random() < 0.5
    if kind == "recurrent":
        t = rng.choice([1, 1, 1, 2, 3, 5, 17])
        b = _log_int(rng, 1, max(1, min(64, 1024 // (h * rep))))
        return {"kind": kind, "B": b, "T": t, "H": h, "HV": h * rep, "K": kd, "V": vd, "gate": gate,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "h0": h0}
    train = rng.random() < 0.5
    tokens = _log_int(rng, 1, min(32768, (262144 if train else 524288) // (h * rep)))
    docs = rng.choice([0, 0, 1]) and rng.randint(1, max(1, min(40, tokens // 2)))
    b = 1 if docs else rng.choice([x for x in (1, 1, 2, 3, 8) if x <= tokens])
    return {"kind": kind, "B": b, "T": max(1, tokens // b), "docs": docs, "H": h, "HV": h * rep, "K": kd, "V": vd,
            "gate": gate, "dtype": "bf16", "h0": h0, "train": train}


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _doc_bounds(total, docs, gen):
    """Bounds of ``docs`` documents of uneven lengths, one token at least each."""
    share = torch.rand(docs, generator=gen).double() + 0.1
    lens = torch.floor(share * (total - docs) / share.sum()).long() + 1
    lens[-1] += total - int(lens.sum())
    return torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)])


def _raw(case, seed):
    """The case's inputs as a dict of tensors on the GPU, without gradients."""
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    dt = DTYPES[case["dtype"]]
    x = {}
    if case["kind"] == "rope":
        b, t, d = case["B"], case["T"], case["D"]
        # column slices of one fused projection's output, as a layer has them
        proj = (randn(b, t, (case["HQ"] + case["HK"]) * d) * 0.7).to(dt)
        x["proj"] = proj
        x["qw"], x["kw"] = 1 + 0.1 * randn(d), 1 + 0.1 * randn(d)
        x["pos"] = None
        if case["pos"]:
            x["pos"] = torch.randint(0, case["pos"], (b, 1), generator=gen, device=DEV) + torch.arange(t, device=DEV)
        if case["train"]:
            x["dq"], x["dk"] = randn(b, t, case["HQ"], d).to(dt), randn(b, t, case["HK"], d).to(dt)
        return x
    b, t, h, hv, kd, vd = (case[n] for n in ("B", "T", "H", "HV", "K", "V"))
    docs = case.get("docs", 0)
    n = docs or b
    x["cu_host"] = _doc_bounds(t, docs, host) if docs else None
    x["cu"] = x["cu_host"].to(DEV) if docs else None
    # q and k as a norm leaves them (unit mean square), v as a projection does
    x["q"], x["k"], x["v"] = randn(b, t, h, kd).to(dt), randn(b, t, h, kd).to(dt), randn(b, t, hv, vd).to(dt)
    if case["gate"] == "token":  # learnt decays: half-lives from a token to a few hundred
        x["g"] = -torch.nn.functional.softplus(randn(b, t, hv)) * torch.exp(
            -1 - 3 * torch.rand(b, t, hv, generator=gen, device=DEV))
    elif case["gate"] == "head":  # one decay a head, 1/2 ... 1/500 a token
        x["g"] = -torch.exp(torch.linspace(math.log(0.5), math.log(0.002), hv, device=DEV) + 0.1 * randn(hv))
    else:
        x["g"] = None
    x["h0"] = randn(n, hv, kd, vd) if case["h0"] else None
    if case.get("train"):
        x["do"] = randn(b, t, hv, vd).to(dt)
        x["dht"] = randn(n, hv, kd, vd) if case["h0"] else None
    return x


def prepare(case, seed):
    x = _raw(case, seed)
    leaves = []
    if case.get("train"):
        for name in ("proj", "qw", "kw") if case["kind"] == "rope" else ("q", "k", "v", "g", "h0"):
            if x[name] is not None:
                x[name].requires_grad_(True)
                leaves.append(name)
    return {"case": case, "x": x, "leaves": leaves}


# ---------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------
def _pad_index(cu, total):
    """[docs, longest] token numbers of packed documents (``total``, one past the end, where a document has none)."""
    lens = cu[1:] - cu[:-1]
    steps = torch.arange(int(lens.max()))
    idx = cu[:-1, None] + steps
    return torch.where(steps < lens[:, None], idx, torch.full_like(idx, total)).to(DEV)


def _plain_attention(q, k, v, g, scale, h0, cu_host):
    """Chunks of 64 tokens: the scores inside a chunk, the state between chunks, 32 bits (decays summed in 64)."""
    b, t, h, kd = q.shape
    hv, vd = v.shape[2], v.shape[3]
    dt = q.dtype
    q, k, v = q.float(), k.float(), v.float()
    g = torch.zeros(b, t, hv, device=q.device) if g is None else g.float().expand(b, t, hv)
    if hv != h:
        q, k = q.repeat_interleave(hv // h, 2), k.repeat_interleave(hv // h, 2)
    idx = None
    if cu_host is not None:
        idx = _pad_index(cu_host, t)

        def pad(x):
            return torch.cat([x[0], torch.zeros_like(x[0, :1])])[idx]

        q, k, v, g = pad(q), pad(k), pad(v), pad(g)
    n, length = q.shape[:2]
    nc = -(-length // CHUNK)
    fill = nc * CHUNK - length

    def chunks(x):  # [n, length, hv, *] -> [n, hv, nc, 64, *]
        x = torch.cat([x, x.new_zeros(n, fill, *x.shape[2:])], 1) if fill else x
        return x.reshape(n, nc, CHUNK, *x.shape[2:]).movedim(3, 1)

    q, k, v, g = chunks(q), chunks(k), chunks(v), chunks(g.double())
    acc = g.cumsum(3)
    causal = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = torch.where(causal, acc[..., :, None] - acc[..., None, :], -math.inf).exp().float()
    o = ((q @ k.transpose(-1, -2).contiguous()) * decay) @ v
    last = acc[..., -1:]
    add = (k * (last - acc).exp().float()[..., None]).transpose(-1, -2).contiguous() @ v
    keep = last.exp().float()[..., None]
    s = h0.float() if h0 is not None else torch.zeros(n, hv, kd, vd, device=q.device)
    entry = []
    for c in range(nc):
        entry.append(s)
        s = s * keep[:, :, c] + add[:, :, c]
    o = scale * (o + (q * acc.exp().float()[..., None]) @ torch.stack(entry, 2))
    o = o.movedim(1, 3).reshape(n, nc * CHUNK, hv, vd)[:, :length]
    if idx is not None:
        o = o[idx < t][None]
    return o.to(dt), s


def _plain_recurrent(q, k, v, g, scale, h0):
    b, t, h, kd = q.shape
    hv, vd = v.shape[2], v.shape[3]
    dt = q.dtype
    q, k, v = q.float(), k.float(), v.float()
    if hv != h:
        q, k = q.repeat_interleave(hv // h, 2), k.repeat_interleave(hv // h, 2)
    a = None if g is None else g.float().exp().expand(b, t, hv)
    s = h0 if h0 is not None else torch.zeros(b, hv, kd, vd, device=q.device)
    out = []
    for i in range(t):
        if a is not None:
            s = s * a[:, i, :, None, None]
        s = s + k[:, i, :, :, None] * v[:, i, :, None, :]
        out.append(scale * (q[:, i, :, :, None] * s).sum(2))
    return torch.stack(out, 1).to(dt), s


def _plain_rope(x, w, pos, rot):
    """RMSNorm of the last axis, then the rotation of its first ``rot`` entries; angles in 64 bits."""
    dt = x.dtype
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    half = rot // 2
    inv = THETA ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    angle = (pos.double()[..., None] * inv)[:, :, None, :]
    cos, sin = angle.cos().float(), angle.sin().float()
    lo, hi = y[..., :half], y[..., half:rot]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, y[..., rot:]], -1).to(dt)


def _rope_views(case, proj):
    b, t, d = case["B"], case["T"], case["D"]
    nq = case["HQ"] * d
    return proj[..., :nq].unflatten(-1, (case["HQ"], d)), proj[..., nq:].unflatten(-1, (case["HK"], d))


def run(state):
    case, x = state["case"], state["x"]
    if case["kind"] == "rope":
        q, k = _rope_views(case, x["proj"])
        if own:
            from sorernn_amd import qk_norm_rope

            out = list(qk_norm_rope(q, k, x["qw"], x["kw"], positions=x["pos"], rot_dim=case["rot"], theta=THETA, eps=EPS))
        else:
            pos = x["pos"]
            if pos is None:
                pos = torch.arange(case["T"], device=DEV).expand(case["B"], case["T"])
            out = [_plain_rope(q, x["qw"], pos, case["rot"]), _plain_rope(k, x["kw"], pos, case["rot"])]
        up = [x["dq"], x["dk"]] if case["train"] else []
    else:
        scale = case["K"] ** -0.5
        if own:
            from sorernn_amd import chunk_decay_linear_attention, fused_recurrent_decay_linear_attention

            if case["kind"] == "chunk":
                out = chunk_decay_linear_attention(x["q"], x["k"], x["v"], x["g"], scale=scale, initial_state=x["h0"],
                                                   output_final_state=True, cu_seqlens=x["cu"],
                                                   cu_seqlens_cpu=x["cu_host"])
            else:
                out = fused_recurrent_decay_linear_attention(x["q"], x["k"], x["v"], x["g"], scale=scale,
                                                             initial_state=x["h0"], output_final_state=True)
        elif case["kind"] == "chunk":
            out = _plain_attention(x["q"], x["k"], x["v"], x["g"], scale, x["h0"], x["cu_host"])
        else:
            out = _plain_recurrent(x["q"], x["k"], x["v"], x["g"], scale, x["h0"])
        out = list(out)
        up = []
        if case.get("train"):
            up = [x["do"]] + ([x["dht"]] if x["dht"] is not None else [])
    if up:
        grads = torch.autograd.grad(out[:len(up)], [x[n] for n in state["leaves"]], up)
        out = [o.detach() for o in out] + list(grads)
    return out


# ---------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------
def _exact_attention(case, x):
    b, t, h, hv, kd, vd = (case[n] for n in ("B", "T", "H", "HV", "K", "V"))
    scale, rep = kd**-0.5, hv // h
    if x.get("cu_host") is not None:
        cu = x["cu_host"].tolist()
        spans = [(0, p, e) for p, e in zip(cu[:-1], cu[1:])]
    else:
        spans = [(i, 0, t) for i in range(b)]
    n, longest = len(spans), max(e - p for _, p, e in spans)

    def rows(y, heads):  # [longest, n, hv, width], zeros behind a sequence's end
        out = torch.zeros(longest, n, hv, y.shape[-1], dtype=torch.float64, device=DEV)
        for i, (bi, p, e) in enumerate(spans):
            out[:e - p, i] = y[bi, p:e].double().repeat_interleave(hv // heads, 1)
        return out

    q, k, v = rows(x["q"], h), rows(x["k"], h), rows(x["v"], hv)
    if x["g"] is None:
        g = torch.zeros(longest, n, hv, dtype=torch.float64, device=DEV)
    else:
        gt = x["g"].detach().double()
        g = rows((gt if gt.dim() == 3 else gt.expand(b, t, hv))[..., None], hv)[..., 0]
    h0 = x["h0"].detach().double() if x["h0"] is not None else torch.zeros(n, hv, kd, vd, dtype=torch.float64, device=DEV)
    a = g.exp()[..., None, None]

    def back(y, heads):  # [longest, n, hv, width] -> [b, t, heads, width]
        out = torch.empty(b, t, heads, y.shape[-1], dtype=torch.float64, device=DEV)
        for i, (bi, p, e) in enumerate(spans):
            out[bi, p:e] = y[:e - p, i].reshape(e - p, heads, hv // heads, -1).sum(2)
        return out

    train = case.get("train", False)
    o, s = torch.empty_like(v), h0.clone()
    if train:
        do, dq = rows(x["do"], hv), torch.empty_like(k)
    for i in range(longest):
        s.mul_(a[i]).add_(k[i, :, :, :, None] * v[i, :, :, None, :])
        o[i] = scale * (q[i, :, :, :, None] * s).sum(2)
        if train:
            dq[i] = scale * (s * do[i, :, :, None, :]).sum(3)
    out = [back(o, hv), s]
    if not train:
        return out
    dht = x["dht"].double() if x["dht"] is not None else torch.zeros_like(s)
    r, dk, dv = dht.clone(), torch.empty_like(k), torch.empty_like(v)
    for i in reversed(range(longest)):
        if i + 1 < longest:
            r.mul_(a[i + 1])
        r.add_(scale * q[i, :, :, :, None] * do[i, :, :, None, :])
        dk[i] = (r * v[i, :, :, None, :]).sum(3)
        dv[i] = (r * k[i, :, :, :, None]).sum(2)
    out += [back(dq, h), back(dk, h), back(dv, hv)]
    if x["g"] is not None:
        each = ((q * dq).sum(3) - (k * dk).sum(3)).flip(0).cumsum(0).flip(0) + (s * dht).sum((2, 3))
        dg = back(each[..., None], hv)[..., 0]
        out.append(dg if x["g"].dim() == 3 else dg.sum((0, 1)))
    if x["h0"] is not None:
        out.append(r * a[0])
    return out


def _exact_rope(case, x):
    b, t, d, rot = case["B"], case["T"], case["D"], case["rot"]
    pos = x["pos"] if x["pos"] is not None else torch.arange(t, device=DEV).expand(b, t)
    freq = torch.tensor([THETA ** (-2.0 * f / rot) for f in range(rot // 2)], dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.ones(b, t, 1, rot // 2, dtype=torch.float64, device=DEV),
                       pos.double()[:, :, None, None] * freq)
    nq = case["HQ"] * d
    outs, grads, wgrads = [], [], []
    proj = x["proj"].detach().double()
    for lo, hi, w, up in ((0, nq, x["qw"], x.get("dq")), (nq, proj.shape[-1], x["kw"], x.get("dk"))):
        w = w.detach().double()
        z = proj[..., lo:hi].reshape(b, t, -1, d)
        r = 1 / torch.sqrt((z * z).sum(-1, keepdim=True) / d + EPS)
        y = z * r * w

        def rotate(m, by):
            c = torch.complex(m[..., :rot // 2].contiguous(), m[..., rot // 2:rot].contiguous()) * by
            return torch.cat([c.real, c.imag, m[..., rot:]], -1)

        outs.append(rotate(y, turn))
        if case["train"]:
            dy = rotate(up.double(), turn.conj())
            wgrads.append((dy * z * r).sum((0, 1, 2)))
            dn = dy * w
            grads.append((r * dn - z * r**3 * (dn * z).sum(-1, keepdim=True) / d).reshape(b, t, hi - lo))
    if case["train"]:
        outs.append(torch.cat(grads, -1))
        outs += wgrads
    return outs


def exact(case, seed):
    x = _raw(case, seed)
    return _exact_rope(case, x) if case["kind"] == "rope" else _exact_attention(case, x)


def work(case):
    b, t, size = case["B"], case["T"], SIZE[case["dtype"]]
    if case["kind"] == "rope":
        elems = b * t * (case["HQ"] + case["HK"]) * case["D"]
        # forward: x read, y written; backward besides: dy read, dx written
        return {"bytes": elems * size * (4 if case["train"] else 2) + case["D"] * 8 * (2 if case["train"] else 1),
                "flops": elems * (24 if case["train"] else 8)}
    h, hv, kd, vd = (case[n] for n in ("H", "HV", "K", "V"))
    n = case.get("docs", 0) or b
    rows = b * t * (2 * h * kd + 2 * hv * vd) * size  # q, k, v and o
    gate = {"token": b * t * hv * 4, "head": hv * 4, "none": 0}[case["gate"]]
    states = n * hv * kd * vd * 4
    flops = 4 * b * t * hv * kd * vd
    total = rows + gate + states * (2 if case["h0"] else 1)
    if case.get("train"):
        total += rows + gate + (states * 2 if case["h0"] else 0)  # do, dq, dk, dv; dg; the states' gradients
        flops *= 3
    return {"bytes": total, "flops": flops}
