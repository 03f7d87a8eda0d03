"""GPU: decay linear attention (chunked with backward, recurrent) and the q/k norm with rotation against 64 bits.

Error bounds, per term of a result's sum (tests/linear_ref.py), u = 2^-24:
- chunked o, dq, dk, dv: scores and states are multiplied as two bf16 parts, off by 2^-16 at most of a term, in two
  places (the state of a chunk and its scores are different terms: one each); sums of up to K + 64 products and the
  states' own error below: 2^-14 in all. Then one rounding to bf16.
- chunked states, dh0: three bf16 parts (u), an exponential (4 u), sums of 64 products a chunk, one product with the
  chunk's or segment's decay for each (2 u each, 20 chunks and 10 segments at most here): (64 + 60 + 5) u < 2^-16.
- dg: the same states, times rows of K + V products, exact scores summed over 64 rows and 64 columns: 2^-15.
- recurrent: T + K sums and T decays: (2 T + K + 8) u.
"""
import pytest
import torch

from sorernn_amd import (chunk_decay_linear_attention, fused_recurrent_decay_linear_attention, qk_norm_rope, rms_norm_gated)
from tests.linear_ref import check, decay_attention, norm_rope

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24
OUT, STATE, GATE = 2.0**-14, 2.0**-16, 2.0**-15


def _cu(lens):
    return torch.cat([torch.zeros(1, dtype=torch.long), torch.tensor(lens).cumsum(0)]) if lens else None


def _inputs(b, t, h, hv, kd, vd, gate="token", h0=False, lens=None, dtype=torch.bfloat16, seed=0, train=False):
    gen = torch.Generator(DEV).manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, generator=gen, device=DEV)

    x = {"q": rnd(b, t, h, kd).to(dtype), "k": rnd(b, t, h, kd).to(dtype), "v": rnd(b, t, hv, vd).to(dtype)}
    g = -torch.nn.functional.softplus(rnd(b, t, hv)) * torch.exp(-3 * torch.rand(b, t, hv, generator=gen, device=DEV))
    if gate == "strong":  # resets now and then, some exact
        g = torch.where(rnd(b, t, hv) > 1.5, torch.full_like(g, -torch.inf), 30 * g)
    elif gate == "growing":
        g = 0.2 * rnd(b, t, hv)
    elif gate == "head":
        g = -torch.rand(hv, generator=gen, device=DEV)
    elif gate == "bf16":
        g = g.bfloat16()
    x["g"] = None if gate == "none" else g
    n = len(lens) if lens else b
    x["h0"] = rnd(n, hv, kd, vd) if h0 else None
    x["cu"] = _cu(lens)
    if train:
        x["do"] = rnd(b, t, hv, vd).to(dtype)
        x["dht"] = rnd(n, hv, kd, vd) if h0 else None
    return x


def _call(fn, x, scale, final=True, **kw):
    cu = None if x["cu"] is None else x["cu"].to(DEV)
    return fn(x["q"], x["k"], x["v"], x["g"], scale=scale, initial_state=x["h0"], output_final_state=final, cu_seqlens=cu,
              cu_seqlens_cpu=x["cu"], **kw)


CASES = [
    # B, T, H, HV, K, V, gate, h0, lens
    (1, 1, 1, 1, 64, 64, "token", True, None),
    (2, 63, 2, 2, 128, 128, "token", False, None),
    (1, 64, 1, 2, 64, 128, "head", True, None),
    (3, 65, 2, 4, 128, 64, "none", True, None),
    (1, 257, 2, 2, 128, 128, "strong", True, None),
    (2, 300, 1, 3, 64, 64, "bf16", False, None),
    (1, 512, 1, 1, 128, 128, "growing", True, None),
    (1, 1281, 1, 2, 128, 128, "token", True, None),
    (1, 1281, 2, 2, 64, 128, "head", False, None),
    (1, 1000, 2, 2, 128, 128, "token", True, [1, 64, 65, 255, 256, 257, 1, 101]),
    (1, 700, 1, 2, 64, 64, "strong", True, [300, 1, 399]),
    (1, 70, 2, 2, 128, 64, "token", True, [3, 2, 65]),
    (1, 330, 1, 1, 64, 128, "none", False, [1] * 130 + [200]),
]
IDS = [f"{c[0]}x{c[1]}-h{c[2]}.{c[3]}-{c[4]}.{c[5]}-{c[6]}{'-h0' if c[7] else ''}{'-docs' if c[8] else ''}" for c in CASES]


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_chunk_forward(case):
    b, t, h, hv, kd, vd, gate, h0, lens = case
    x = _inputs(b, t, h, hv, kd, vd, gate, h0, lens)
    scale = kd**-0.5
    o, s = _call(chunk_decay_linear_attention, x, scale)
    ref = decay_attention(x["q"], x["k"], x["v"], x["g"], scale, x["h0"], x["cu"])
    assert o.dtype == torch.bfloat16 and s.dtype == torch.float32
    check(o, ref, "o", OUT)
    check(s, ref, "state", STATE)
    o2, none = _call(chunk_decay_linear_attention, x, scale, final=False)
    assert none is None and torch.equal(o, o2)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_chunk_backward(case):
    b, t, h, hv, kd, vd, gate, h0, lens = case
    x = _inputs(b, t, h, hv, kd, vd, gate, h0, lens, train=True)
    scale = -0.3  # a factor of either sign
    leaves = [n for n in ("q", "k", "v", "g", "h0") if x[n] is not None]
    for n in leaves:
        x[n].requires_grad_(True)
    o, s = _call(chunk_decay_linear_attention, x, scale)
    outs, ups = ([o, s], [x["do"], x["dht"]]) if h0 else ([o], [x["do"]])
    grads = dict(zip(leaves, torch.autograd.grad(outs, [x[n] for n in leaves], ups)))
    with torch.no_grad():
        ref = decay_attention(x["q"], x["k"], x["v"], x["g"], scale, x["h0"], x["cu"], x["do"], x["dht"])
    check(grads["q"], ref, "dq", OUT)
    check(grads["k"], ref, "dk", OUT)
    check(grads["v"], ref, "dv", OUT)
    if h0:
        check(grads["h0"], ref, "dh0", STATE)
    if gate == "head":
        ref["dg"], ref["dg_mag"] = ref["dg"].sum((0, 1)), ref["dg_mag"].sum((0, 1))
    if gate != "none":
        # -inf is a constant: the formula's gradient there is exp(g) <S, R> = 0
        if gate == "strong":
            at = x["g"].detach() == -torch.inf
            ref["dg"] = torch.where(at, torch.zeros_like(ref["dg"]), ref["dg"])
        # the sum over tokens of an expanded gate adds t roundings
        check(grads["g"], ref, "dg", GATE + (t * U if gate == "head" else 0))


def test_chunk_gradients_against_differences():
    x = _inputs(1, 320, 1, 2, 64, 64, "token", True, train=True, seed=3)
    scale = 64**-0.5
    names = ["q", "k", "v", "g", "h0"]
    for n in names:
        x[n].requires_grad_(True)
    o, s = _call(chunk_decay_linear_attention, x, scale)
    grads = torch.autograd.grad([o, s], [x[n] for n in names], [x["do"], x["dht"]])

    def loss(args):
        r = decay_attention(args["q"], args["k"], args["v"], args["g"], scale, args["h0"], None)
        return ((r["o"] * x["do"].double()).sum() + (r["state"] * x["dht"].double()).sum()).item()

    gen = torch.Generator(DEV).manual_seed(5)
    with torch.no_grad():
        for n, grad in zip(names, grads):
            way = torch.randn(x[n].shape, generator=gen, device=DEV, dtype=torch.float64)
            eps = 1e-5
            ends = [loss({m: (x[m].double() + (c * eps * way if m == n else 0)) for m in names}) for c in (1, -1)]
            diff = (ends[0] - ends[1]) / (2 * eps)
            terms = grad.double() * way
            # the gradient's own rounding, by half a step each, and the second difference's share of g's third order
            assert abs(terms.sum().item() - diff) <= 2.0**-8 * terms.abs().sum().item() + 1e-6 * abs(diff), n


def test_chunk_same_bits_twice_and_alone():
    """No atomics: two runs agree bit for bit, and a document alone agrees with itself among others."""
    x = _inputs(1, 700, 2, 4, 128, 128, "token", True, [300, 1, 399], train=True)
    leaves = ["q", "k", "v", "g", "h0"]
    for n in leaves:
        x[n].requires_grad_(True)
    runs = []
    for _ in range(2):
        o, s = _call(chunk_decay_linear_attention, x, 0.1)
        runs.append([o, s, *torch.autograd.grad([o, s], [x[n] for n in leaves], [x["do"], x["dht"]])])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_chunk_no_tokens_and_no_gradient():
    x = _inputs(2, 0, 1, 1, 64, 64, "token", True)
    o, s = _call(chunk_decay_linear_attention, x, 1.0)
    assert o.shape == (2, 0, 1, 64) and torch.equal(s, x["h0"])
    x["h0"].requires_grad_(True)
    o, s = _call(chunk_decay_linear_attention, x, 1.0)
    up = torch.randn_like(s)
    (d,) = torch.autograd.grad(s, [x["h0"]], up)
    assert torch.equal(d, up)
    o, s = _call(fused_recurrent_decay_linear_attention, {**x, "h0": x["h0"].detach()}, 1.0)
    assert torch.equal(s, x["h0"].detach())


def test_chunk_only_the_state_has_a_gradient():
    x = _inputs(1, 300, 1, 1, 64, 64, "token", True, train=True)
    for n in ("q", "k", "v", "g"):
        x[n].requires_grad_(True)
    _, s = _call(chunk_decay_linear_attention, x, 0.2)
    got = torch.autograd.grad(s, [x[n] for n in ("q", "k", "v", "g")], x["dht"])
    with torch.no_grad():
        ref = decay_attention(x["q"], x["k"], x["v"], x["g"], 0.2, x["h0"], None, torch.zeros_like(x["do"]), x["dht"])
    assert not got[0].any()
    for n, y in zip(("dk", "dv", "dg"), got[1:]):
        check(y, ref, n, GATE if n == "dg" else OUT)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_chunk_non_finite_token_leaves_others_alone(which, bad):
    """A token's infinity or NaN reaches it and the tokens after it (q: it alone), in its chunk as in others."""
    x = _inputs(1, 200, 1, 1, 128, 128, "token", True)
    clean, _ = _call(chunk_decay_linear_attention, x, 0.1)
    x[which] = x[which].clone()
    x[which][0, 100, 0, 5] = bad
    o, s = _call(chunk_decay_linear_attention, x, 0.1)
    assert torch.equal(o[:, :64], clean[:, :64])  # the chunks before run as they did
    ref = decay_attention(*(x[n].nan_to_num(0, 0, 0) for n in ("q", "k", "v")), x["g"], 0.1, x["h0"])
    check(o[:, :100], {"o": ref["o"][:, :100], "o_mag": ref["o_mag"][:, :100]}, "o", OUT)
    assert not torch.isfinite(o[:, 100].float()).all()
    if which == "q":
        assert torch.equal(o[:, 101:], clean[:, 101:]) and torch.isfinite(s).all()
    else:
        assert not torch.isfinite(s).all()


@pytest.mark.parametrize("how", ["whole", "cut", "docs"])
def test_chunk_gate_gradient_without_the_states_gradient(how):
    """An initial state that needs no gradient: its product with the gradient is not known at the sequence's start."""
    t, lens = {"whole": (200, None), "cut": (1500, None), "docs": (1500, [700, 1, 799])}[how]
    x = _inputs(1, t, 1, 2, 64, 128, "token", True, lens, train=True, seed=11)
    x["g"].requires_grad_(True)
    o, s = _call(chunk_decay_linear_attention, x, 0.2)
    (dg,) = torch.autograd.grad([o, s], [x["g"]], [x["do"], x["dht"]])
    with torch.no_grad():
        check(dg, decay_attention(x["q"], x["k"], x["v"], x["g"], 0.2, x["h0"], x["cu"], x["do"], x["dht"]), "dg", GATE)


@pytest.mark.parametrize("t", [200, 1500])
def test_chunk_non_finite_gradient_leaves_later_tokens_alone(t):
    x = _inputs(1, t, 1, 1, 64, 64, "token", True, train=True, seed=12)
    names, at = ["q", "k", "v", "g", "h0"], t // 2
    for n in names:
        x[n].requires_grad_(True)
    o, s = _call(chunk_decay_linear_attention, x, 0.2)
    up = x["do"].clone()
    up[0, at, 0, 3] = float("nan")
    got = torch.autograd.grad([o, s], [x[n] for n in names], [up, x["dht"]])
    with torch.no_grad():
        ref = decay_attention(x["q"], x["k"], x["v"], x["g"], 0.2, x["h0"], None, x["do"], x["dht"])
    for n, y, per in zip(("dq", "dk", "dv", "dg"), got, (OUT, OUT, OUT, GATE)):
        check(y[:, at + 1:], {m: ref[m][:, at + 1:] for m in (n, n + "_mag")}, n, per)
        assert torch.isnan(y[:, at].float()).any()
    assert torch.isnan(got[4]).any()


def test_chunk_gate_gradient_over_a_long_segment():
    """dg is a running sum of differences of dot products D. Rounded at random, each is off by 1.6 u of its root mean square
    (the state 0.8 u, the products' sum 0.9 u, weights 1 u, for either of the two): 2 u; over 1,024 tokens whose sum is known
    at both ends that grows to sqrt(1024 / 6) of it in the mean."""
    x = _inputs(1, 2048, 128, 128, 64, 64, "token", False, train=True, seed=13)
    x["g"].requires_grad_(True)
    o, _ = _call(chunk_decay_linear_attention, x, 0.125, final=False)
    (dg,) = torch.autograd.grad(o, [x["g"]], x["do"])
    with torch.no_grad():
        ref = decay_attention(x["q"], x["k"], x["v"], x["g"], 0.125, None, None, x["do"])["dg"]
        err = (dg.double() - ref).square().mean().sqrt().item()
        assert err <= 2 * U * (1024 / 6)**0.5 * ref.diff(dim=1).square().mean().sqrt().item()


def test_chunk_strided_and_unaligned_inputs():
    x = _inputs(2, 130, 2, 2, 64, 64, "token", True, seed=2)
    want = _call(chunk_decay_linear_attention, x, 0.1)
    y = dict(x)
    y["q"] = x["q"].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(2, 130, 2, 80, device=DEV, dtype=torch.bfloat16)
    wide[..., 3:67] = x["k"]
    y["k"] = wide[..., 3:67]
    flat = torch.zeros(x["v"].numel() + 1, device=DEV, dtype=torch.bfloat16)
    flat[1:] = x["v"].flatten()
    y["v"] = flat[1:].view(x["v"].shape)
    y["g"] = x["g"].transpose(0, 1).contiguous().transpose(0, 1)
    y["h0"] = x["h0"].transpose(2, 3).contiguous().transpose(2, 3)
    for a, b in zip(want, _call(chunk_decay_linear_attention, y, 0.1)):
        assert torch.equal(a, b)
    for a, b in zip(want, _call(chunk_decay_linear_attention, {**x, "h0": x["h0"].double()}, 0.1)):
        assert torch.equal(a, b)


REC = [
    (1, 1, 1, 1, 64, 64, "token", True, None),
    (3, 1, 2, 4, 128, 128, "head", True, None),
    (2, 17, 1, 2, 64, 128, "none", False, None),
    (1, 40, 2, 2, 128, 64, "strong", True, [1, 16, 17, 6]),
    (1, 130, 1, 1, 128, 128, "bf16", False, None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", REC, ids=[f"{c[0]}x{c[1]}-{c[4]}.{c[5]}-{c[6]}" for c in REC])
def test_recurrent(case, dtype):
    b, t, h, hv, kd, vd, gate, h0, lens = case
    x = _inputs(b, t, h, hv, kd, vd, gate, h0, lens, dtype)
    scale = kd**-0.5
    o, s = _call(fused_recurrent_decay_linear_attention, x, scale)
    ref = decay_attention(x["q"], x["k"], x["v"], x["g"], scale, x["h0"], x["cu"])
    per = (2 * t + kd + 8) * U
    check(o, ref, "o", per)
    check(s, ref, "state", per)
    if dtype == torch.float32:  # the chunked operator's route for it
        for a, y in zip((o, s), _call(chunk_decay_linear_attention, x, scale)):
            assert torch.equal(a, y)
    if h0:
        state = x["h0"].clone()
        o2, s2 = _call(fused_recurrent_decay_linear_attention, {**x, "h0": state}, scale, inplace_final_state=True)
        assert s2.data_ptr() == state.data_ptr() and torch.equal(s2, s) and torch.equal(o2, o)


def test_recurrent_continues_a_prompt():
    x = _inputs(2, 300, 2, 4, 128, 128, "token", True)
    n = 290
    cut = {**x, **{m: x[m][:, :n] for m in ("q", "k", "v", "g")}}
    _, state = _call(chunk_decay_linear_attention, cut, 0.1)
    outs = []
    for i in range(n, 300):
        o, state = fused_recurrent_decay_linear_attention(*(x[m][:, i:i + 1] for m in ("q", "k", "v", "g")), scale=0.1,
                                                          initial_state=state, inplace_final_state=True)
        outs.append(o)
    ref = decay_attention(x["q"], x["k"], x["v"], x["g"], 0.1, x["h0"])
    check(torch.cat(outs, 1), {"o": ref["o"][:, n:], "o_mag": ref["o_mag"][:, n:]}, "o", OUT)
    check(state, ref, "state", STATE + 30 * U)


# ---------------------------------------------------------------------------------------------------
# The norm with rotation, per term: a row's sum of squares (D products: D u / 2 through the root), root and quotient (2 u
# each), the products (4 u), an angle rounded to 2^-25 turns (2 pi 2^-25 < 4 u) and a sine (4 u): (D / 2 + 20) u; the
# backward's dot product adds D u and the squares of the same factors: (3 D + 60) u; a weight's sum adds at most as many
# roundings as there are rows for a workgroup.
ROPE = [
    # B, T, HQ, HK, D, rot, positions
    (1, 1, 1, 1, 64, 16, "far"),
    (2, 5, 3, 1, 128, 128, None),
    (3, 7, 4, 4, 256, 256, "shared"),
    (1, 129, 2, 1, 128, 32, "docs"),
    (2, 33, 5, 2, 64, 0, None),
    (64, 1, 8, 2, 128, 64, "far32"),
    (2, 2051, 1, 2, 64, 64, None),
]


def _rope_inputs(case, dtype, seed=0):
    b, t, hq, hk, d, rot, how = case
    gen = torch.Generator(DEV).manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, generator=gen, device=DEV)

    q, k = rnd(b, t, hq, d).to(dtype), (3 * rnd(b, t, hk, d)).to(dtype)
    pos, cu, given = torch.arange(t, device=DEV).expand(b, t), None, None
    if how in ("far", "far32"):
        given = pos = torch.randint(0, 10**6, (b, t), generator=gen, device=DEV)
        given = given.int() if how == "far32" else given
    elif how == "shared":
        given = torch.arange(t, device=DEV) * 1001 + 10**5
        pos = given.expand(b, t)
    elif how == "docs":
        cu = torch.tensor([0, 1, 65, t])
        pos = torch.cat([torch.arange(int(n), device=DEV) for n in cu.diff()])[None]
    return q, k, 1 + 0.2 * rnd(d), 1 + 0.2 * rnd(d), pos, given, cu, rnd(b, t, hq, d).to(dtype), rnd(b, t, hk, d).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", ROPE, ids=[f"{c[0]}x{c[1]}-h{c[2]}.{c[3]}-{c[4]}.{c[5]}" for c in ROPE])
def test_norm_rope(case, dtype):
    b, t, hq, hk, d, rot, _ = case
    q, k, qw, kw, pos, given, cu, uq, uk = _rope_inputs(case, dtype)
    for x in (q, k, qw, kw):
        x.requires_grad_(True)
    theta, eps = 1e4, 1e-6
    out = qk_norm_rope(q, k, qw, kw, given, rot, theta, eps, cu_seqlens=None if cu is None else cu.to(DEV),
                       cu_seqlens_cpu=cu)
    grads = torch.autograd.grad(out, [q, k, qw, kw], [uq, uk])
    with torch.no_grad():
        for x, w, up, y, dx, dw in ((q, qw, uq, out[0], grads[0], grads[2]), (k, kw, uk, out[1], grads[1], grads[3])):
            ref = norm_rope(x, w, pos, rot, theta, eps, up)
            assert y.is_contiguous() and y.dtype == dtype
            check(y.detach(), ref, "y", (d / 2 + 20) * U)
            check(dx, ref, "dx", (3 * d + 60) * U)
            check(dw, ref, "dw", (d / 2 + 40 + b * t * x.shape[2] / 8 + 64) * U)
        bare = qk_norm_rope(q, k, None, None, given, rot, theta, eps, cu_seqlens=None if cu is None else cu.to(DEV),
                            cu_seqlens_cpu=cu)
        check(bare[0], norm_rope(q, None, pos, rot, theta, eps), "y", (d / 2 + 20) * U)


def test_norm_rope_views_of_a_projection():
    gen = torch.Generator(DEV).manual_seed(1)
    proj = torch.randn(2, 9, 6 * 128, generator=gen, device=DEV).bfloat16()
    q, k = proj[..., :512].unflatten(-1, (4, 128)), proj[..., 512:].unflatten(-1, (2, 128))
    want = qk_norm_rope(q.contiguous(), k.contiguous(), rot_dim=32)
    for a, y in zip(want, qk_norm_rope(q, k, rot_dim=32)):
        assert torch.equal(a, y)
    one = proj[:, :, :128].unflatten(-1, (1, 128)).expand(2, 9, 4, 128)  # a broadcast head
    ref = qk_norm_rope(one.contiguous(), k.contiguous(), rot_dim=32)
    for a, y in zip(ref, qk_norm_rope(one, k.transpose(0, 1).contiguous().transpose(0, 1), rot_dim=32)):
        assert torch.equal(a, y)
    odd = torch.zeros(2, 9, 4, 131, device=DEV, dtype=torch.bfloat16)
    odd[..., 1:129] = q
    assert torch.equal(qk_norm_rope(odd[..., 1:129], k, rot_dim=32)[0], want[0])


def test_norm_rope_zero_rows_and_gradient_of_a_broadcast_head():
    q = torch.zeros(1, 3, 2, 64, device=DEV, dtype=torch.bfloat16)
    k = torch.randn(1, 3, 1, 64, device=DEV).bfloat16().requires_grad_(True)
    a, y = qk_norm_rope(q, k.expand(1, 3, 4, 64), rot_dim=64)
    assert not a.any()
    up = torch.randn_like(y)
    (dk,) = torch.autograd.grad(y, [k], up)
    pos = torch.arange(3, device=DEV)[None]
    with torch.no_grad():
        ref = norm_rope(k.expand(1, 3, 4, 64), None, pos, 64, 1e7, 1e-6, up)
        # each of 4 gradients is rounded to bf16 before autograd's sum over the heads, which rounds 3 times more
        r = {"dx": ref["dx"].sum(2, keepdim=True), "dx_mag": ref["dx_mag"].sum(2, keepdim=True)}
    check(dk, r, "dx", 4 * 2.0**-8 + 300 * U)


def test_norm_rope_no_tokens():
    q = torch.zeros(2, 0, 2, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    a, b = qk_norm_rope(q, q, w, w)
    dq, dw = torch.autograd.grad([a.sum() + b.sum()], [q, w])
    assert a.shape == q.shape and dq.shape == q.shape and not dw.any()


# ---------------------------------------------------------------------------------------------------
# together, as a layer has them
# ---------------------------------------------------------------------------------------------------
def _block(x, p, cu=None, cu_host=None, state=None, step=False, positions=None):
    b, t, _ = x.shape
    proj = torch.nn.functional.linear(x, p["w"])
    q, k, v, gate = proj.split([256, 128, 256, 256], -1)
    q, k = qk_norm_rope(q.unflatten(-1, (2, 128)), k.unflatten(-1, (1, 128)).expand(b, t, 2, 128), p["qw"], p["kw"],
                        positions, 32, 1e4, cu_seqlens=cu, cu_seqlens_cpu=cu_host)
    fn = fused_recurrent_decay_linear_attention if step else chunk_decay_linear_attention
    o, s = fn(q, k, v.unflatten(-1, (2, 128)), p["g"], initial_state=state, output_final_state=True, cu_seqlens=cu,
              cu_seqlens_cpu=cu_host)
    y = rms_norm_gated(o, gate.unflatten(-1, (2, 128)), p["ow"], None, activation="swish")
    return torch.nn.functional.linear(y.flatten(-2), p["wo"]), s


def _block_params(seed=0):
    gen = torch.Generator(DEV).manual_seed(seed)

    def rnd(*s, scale=1.0):
        return scale * torch.randn(*s, generator=gen, device=DEV)

    return {"w": rnd(896, 192, scale=0.07).bfloat16(), "wo": rnd(192, 256, scale=0.06).bfloat16(), "qw": 1 + rnd(128, scale=0.1),
            "kw": 1 + rnd(128, scale=0.1), "ow": 1 + rnd(128, scale=0.1), "g": -torch.tensor([0.05, 0.4], device=DEV)}


def test_block_prompt_then_single_tokens_and_training():
    """Norm and rotation, the attention, the gated norm: a prompt and the tokens after it give what the whole text gives
    in one call, and a training step gives every parameter a finite gradient."""
    p = _block_params()
    x = torch.randn(2, 310, 192, device=DEV, generator=torch.Generator(DEV).manual_seed(4)).bfloat16()
    with torch.no_grad():
        whole, s_all = _block(x, p)
        y, s = _block(x[:, :300], p)
        parts = [y]
        for i in range(300, 310):
            y, s = _block(x[:, i:i + 1], p, state=s, step=True, positions=torch.full((2, 1), i, device=DEV))
            parts.append(y)
    # two orders of the same sums before a rounding to bf16 in each of four stages: a few steps of the largest value
    got = torch.cat(parts, 1).double()
    assert (got - whole.double()).norm() <= 8 * 2.0**-8 * whole.double().norm()
    assert (s.double() - s_all.double()).norm() <= 2.0**-8 * s_all.double().norm()
    for w in p.values():
        w.requires_grad_(True)
    y, _ = _block(x, p)
    grads = torch.autograd.grad(y.float().square().mean(), list(p.values()))
    for name, gr in zip(p, grads):
        assert torch.isfinite(gr.float()).all() and gr.any(), name


def test_block_documents_as_alone():
    p = _block_params(1)
    lens = [5, 300, 64]
    x = torch.randn(1, sum(lens), 192, device=DEV, generator=torch.Generator(DEV).manual_seed(6)).bfloat16()
    cu = _cu(lens)
    with torch.no_grad():
        y, s = _block(x, p, cu.to(DEV), cu)
        for i, (a, e) in enumerate(zip(cu[:-1].tolist(), cu[1:].tolist())):
            yi, si = _block(x[:, a:e], p)
            assert (y[:, a:e].double() - yi.double()).norm() <= 2.0**-7 * yi.double().norm()
            assert (s[i:i + 1].double() - si.double()).norm() <= 2.0**-7 * si.double().norm()


# ---------------------------------------------------------------------------------------------------
# streams, graphs, compile
# ---------------------------------------------------------------------------------------------------
def test_two_streams_at_once():
    xs = [_inputs(1, 700, 2, 2, 128, 128, "token", True, seed=s) for s in (1, 2)]
    want = [_call(chunk_decay_linear_attention, x, 0.1) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, st in zip(xs, streams):
        with torch.cuda.stream(st):
            got.append([_call(chunk_decay_linear_attention, x, 0.1) for _ in range(3)])
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(w, o))


def test_graph_replays_of_the_forward_and_a_step():
    x = _inputs(2, 600, 2, 4, 128, 128, "token", True, seed=8)
    cuq = {m: x[m].clone() for m in ("q", "k", "v", "g")}
    w = torch.ones(128, device=DEV)
    pos = torch.full((2, 600), 7, device=DEV)

    def run(d):
        q, k = qk_norm_rope(d["q"], d["k"], w, w, pos, 64)
        o, s = chunk_decay_linear_attention(q, k, d["v"], d["g"], 0.1, x["h0"], True)
        o1, s1 = fused_recurrent_decay_linear_attention(q[:, :1], k[:, :1], d["v"][:, :1], d["g"][:, :1], 0.1, s, True)
        return o, s, o1, s1

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(cuq)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(cuq)
    for seed in (8, 9, 10):
        y = _inputs(2, 600, 2, 4, 128, 128, "token", True, seed=seed)
        for m in cuq:
            cuq[m].copy_(y[m])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, run(y)):
            assert torch.equal(a, b)


def test_graph_of_documents_takes_other_lengths():
    """What a captured call launches depends on the number of tokens and documents alone."""
    first, lens = [300, 1, 399], [[300, 1, 399], [64, 635, 1], [1, 1, 698]]
    x = _inputs(1, 700, 2, 4, 128, 64, "token", True, first, seed=14, train=True)
    cu, leaves = x["cu"].to(DEV), ["q", "k", "v", "g", "h0"]

    def step(cu_dev, host):
        a = {m: x[m].detach().requires_grad_(True) for m in leaves}
        q, k = qk_norm_rope(a["q"], a["k"], rot_dim=32, cu_seqlens=cu_dev, cu_seqlens_cpu=host)
        o, s = chunk_decay_linear_attention(q, k, a["v"], a["g"], 0.1, a["h0"], True, cu_dev, host)
        grads = torch.autograd.grad([o, s], [a[m] for m in leaves], [x["do"], x["dht"]])
        with torch.no_grad():
            o2, s2 = fused_recurrent_decay_linear_attention(q, k, a["v"], a["g"], 0.1, s, True, cu_seqlens=cu_dev,
                                                            cu_seqlens_cpu=host)
        return [o, s, *grads, o2, s2]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(cu, x["cu"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(cu, x["cu"])
    for n in lens:
        now = _cu(n)
        cu.copy_(now)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step(now.to(DEV), now)):
            assert torch.equal(a, b)


def test_compiled_for_any_length():
    """One compiled function over lengths on both sides of the split, with documents and their states."""
    def f(q, k, v, g, h0, cu):
        q, k = qk_norm_rope(q, k, rot_dim=32, cu_seqlens=cu)
        return chunk_decay_linear_attention(q, k, v, g, 0.1, h0, True, cu)

    torch._dynamo.reset()
    compiled = torch.compile(f, fullgraph=True, dynamic=True, backend="aot_eager")
    for lens in ([60, 40], [300, 500], [1000, 37]):
        x = _inputs(1, sum(lens), 1, 2, 64, 128, "token", True, lens, train=True, seed=17)
        outs = []
        for fn in (f, compiled):
            a = [x[m].detach().requires_grad_(True) for m in ("q", "k", "v", "g", "h0")]
            o, s = fn(*a, x["cu"].to(DEV))
            outs.append([o, s, *torch.autograd.grad([o, s], a, [x["do"], x["dht"]])])
        for a, b in zip(*outs):
            assert torch.equal(a, b)
    torch._dynamo.reset()


@pytest.mark.parametrize("bounds, docs", [
    ([0, 300, 301, 650], [(0, 300), (300, 301), (301, 650)]),  # rows behind the last document
    ([0, 64, 64, 699], [(0, 64), (64, 699)]),                  # an empty document
    ([130, 131, 131, 5000], [(130, 131), (131, 700)]),         # rows before the first one, an end past the tokens
    ([-7, 0, 0, 0], []),
    ([0, 650, 300, 700], None),                                # out of order
])
def test_bounds_that_no_call_checked(bounds, docs):
    """Captured and compiled calls take the documents' bounds as they are. In ascending order the documents come out right
    and other tokens stay as they were; whatever the bounds hold, nothing outside the tensors is written."""
    from sorernn_amd import _lib, linear

    x = _inputs(1, 700, 1, 2, 64, 64, "token", True, [300, 1, 399], seed=16, train=True)
    cu = torch.tensor(bounds, device=DEV)
    wide = torch.full((5, 2, 64, 64), 7.0, device=DEV)
    o = torch.full((3, 700, 2, 64), 7.0, device=DEV, dtype=torch.bfloat16)
    need = _lib.load().gdn_decay_attn_states_size(1, 700, 2, 64, 64, 3, 1)
    states = torch.full((need + 256,), 3, device=DEV, dtype=torch.uint8)
    _lib.call("gdn_decay_attn_fwd", x["q"].data_ptr(), x["k"].data_ptr(), x["v"].data_ptr(), x["g"].data_ptr(),
              x["h0"].data_ptr(), o[1].data_ptr(), wide[1].data_ptr(), cu.data_ptr(), 1, 700, 1, 2, 64, 64, 3, 0,
              *x["g"].stride(), 0.1, 0, states.data_ptr(), need, _lib.stream_of(o))
    grads = linear.attention_bwd_impl(x["q"], x["k"], x["v"], x["g"], x["h0"], None, x["do"], None, states[:need], cu, 0.1, 0, 3,
                                      True, True)
    rec = torch.full((3, 700, 2, 64), 7.0, device=DEV, dtype=torch.bfloat16)
    _lib.call("gdn_decay_attn_recurrent_fwd", x["q"].data_ptr(), x["k"].data_ptr(), x["v"].data_ptr(), x["g"].data_ptr(), None,
              rec[1].data_ptr(), None, cu.data_ptr(), 1, 700, 1, 2, 64, 64, 3, 1, 0, *x["g"].stride(), 0.1, 0,
              _lib.stream_of(o))
    torch.cuda.synchronize()
    for y in (wide[0], wide[4], o[0], o[2], rec[0], rec[2]):
        assert bool((y == 7).all())
    assert bool((states[need:] == 3).all())
    inside = torch.zeros(700, dtype=torch.bool, device=DEV)
    for a, e in docs or []:
        inside[a:e] = True
        n = max(i for i in range(3) if bounds[i] <= a)  # the last of those that begin there
        part = {m: x[m][:, a:e] for m in ("q", "k", "v", "g", "do")}
        ref = decay_attention(*(part[m] for m in ("q", "k", "v", "g")), 0.1, x["h0"][n:n + 1], None, part["do"])
        check(o[1:2, a:e], ref, "o", OUT)
        for name, y in zip(("dq", "dk", "dv", "dg"), grads):
            check(y[:, a:e], ref, name, GATE if name == "dg" else OUT)
    assert docs is None or bool((o[1][~inside] == 7).all() and (rec[1][~inside] == 7).all())


def test_elements_past_32_bits():
    """2^31 and more elements a tensor. The inputs repeat every 1,024 tokens and a weight of e^-100 is nothing beside the
    others, so tokens 1,024 apart have the same results: two roundings of them apart."""
    t, h, d, back = 2**20 + 700, 16, 128, 1024 * 1000
    x = _inputs(1, 1024, h, h, d, d, "token", False, train=True, seed=15)
    reps = t // 1024 + 1
    big = {m: x[m].repeat(1, reps, 1, 1)[:, :t].contiguous() for m in ("q", "k", "v", "do")}
    assert big["q"].numel() > 2**31
    g = torch.full((h,), -1.0, device=DEV, requires_grad=True).expand(1, t, h)
    for m in ("q", "k", "v"):
        big[m].requires_grad_(True)
    o, s = chunk_decay_linear_attention(big["q"], big["k"], big["v"], g, 0.1, output_final_state=True)
    got = [o, *torch.autograd.grad(o, [big["q"], big["k"], big["v"], g], big["do"])]
    assert torch.isfinite(s).all()
    for y in got:
        late, early = (y[:, a:a + 400].detach().double() for a in (t - 1000, t - 1000 - back))
        assert late.any() and (late - early).norm() <= 2.0**-8 * early.norm()
    del got, o, y
    with torch.no_grad():
        a, _ = qk_norm_rope(big["q"], big["k"], rot_dim=64)
        want, _ = qk_norm_rope(big["q"][:, -300:], big["k"][:, -300:], rot_dim=64,
                               positions=torch.arange(t - 300, t, device=DEV))
        assert torch.equal(a[:, -300:], want)


def test_graph_of_a_training_step():
    x = _inputs(2, 300, 1, 2, 64, 128, "token", False, seed=8, train=True)
    leaves = ["q", "k", "v", "g"]

    def step(d):
        a = [d[m].detach().requires_grad_(True) for m in leaves]
        w = torch.ones(64, device=DEV, requires_grad=True)
        q, k = qk_norm_rope(a[0], a[1], w, w, rot_dim=32)
        o, _ = chunk_decay_linear_attention(q, k, a[2], a[3], 0.1)
        return torch.autograd.grad(o, [*a, w], d["do"])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.synchronize()
    static = {m: x[m].clone() for m in (*leaves, "do")}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for seed in (8, 9, 10):
        y = _inputs(2, 300, 1, 2, 64, 128, "token", False, seed=seed, train=True)
        for m in static:
            static[m].copy_(y[m])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step(y)):
            assert torch.equal(a, b)


def test_compiled_step_has_one_graph_and_the_same_values():
    x = _inputs(1, 300, 1, 2, 64, 64, "head", False, train=True)
    w = torch.ones(64, device=DEV)

    def f(q, k, v, g):
        q, k = qk_norm_rope(q, k, w, w, rot_dim=32)
        return chunk_decay_linear_attention(q, k, v, g, 0.1)[0]

    outs = []
    for fn in (f, torch.compile(f, fullgraph=True, backend="aot_eager")):
        a = [x[m].detach().requires_grad_(True) for m in ("q", "k", "v", "g")]
        o = fn(*a)
        outs.append([o, *torch.autograd.grad(o, a, x["do"])])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_rows_behind_the_outputs_stay_as_they_were():
    """A ragged call writes its rows, its states and nothing beside them."""
    from sorernn_amd import _lib

    x = _inputs(1, 67, 1, 1, 64, 64, "token", False)
    want, state = _call(chunk_decay_linear_attention, x, 0.1)
    o = torch.full((3, 67, 64), 7.0, device=DEV, dtype=torch.bfloat16)
    s = torch.full((3, 64, 64), 7.0, device=DEV)
    _lib.call("gdn_decay_attn_fwd", x["q"].data_ptr(), x["k"].data_ptr(), x["v"].data_ptr(), x["g"].data_ptr(), None,
              o[1].data_ptr(), s[1].data_ptr(), None, 1, 67, 1, 1, 64, 64, 1, 0, *x["g"].stride(), 0.1, 0, None, 0,
              _lib.stream_of(o))
    torch.cuda.synchronize()
    assert torch.equal(o[1], want[0, :, 0]) and torch.equal(s[1], state[0, 0])
    for y in (o[0], o[2], s[0], s[2]):
        assert bool((y == 7).all())
