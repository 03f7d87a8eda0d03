"""GPU: the decay linear attention's values where a call is cut into segments and where types meet."""
import pytest
import torch

from sorernn_amd import chunk_decay_linear_attention, qk_norm_rope
from tests.test_gpu_linear import DEV, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("t", [200, 2000], ids=["whole", "cut"])
def test_non_finite_token_stays_over_segments_that_decay_to_nothing(t, bad):
    """exp(-256) over a segment's 128 tokens is 0 in fp32, and 0 times an infinity or NaN is NaN: how a call is cut does not
    decide whether a bad token shows behind it (its column) and, in the backward, before it."""
    x = _inputs(1, t, 1, 1, 64, 64, "none", True, train=True, seed=31)
    x["v"][0, 10, 0, 5] = bad
    g = torch.full((1,), -2.0, device=DEV)
    o, s = chunk_decay_linear_attention(x["q"], x["k"], x["v"], g, 0.2, x["h0"], True)
    assert not torch.isfinite(o[0, 10:, 0, 5].float()).any() and not torch.isfinite(s[..., 5]).any()
    rest = [c for c in range(64) if c != 5]
    assert torch.isfinite(o[..., rest].float()).all() and torch.isfinite(s[..., rest]).all()
    assert torch.isfinite(o[:, :10].float()).all()

    y = _inputs(1, t, 1, 1, 64, 64, "none", True, train=True, seed=31)
    names = ("q", "k", "v", "h0")
    for n in names:
        y[n].requires_grad_(True)
    o, s = chunk_decay_linear_attention(y["q"], y["k"], y["v"], g, 0.2, y["h0"], True)
    up = y["do"].clone()
    up[0, t - 10, 0, 3] = bad
    dq, dk, dv, dh0 = torch.autograd.grad([o, s], [y[n] for n in names], [up, y["dht"]])
    assert not torch.isfinite(dv[0, :t - 9, 0, 3].float()).any() and not torch.isfinite(dh0[..., 3]).any()
    assert not torch.isfinite(dk[0, :t - 9].float()).any()
    for z in (dq, dk, dv):
        assert torch.isfinite(z[:, t - 9:].float()).all()


def test_norm_rope_of_one_padded_row():
    wide = torch.randn(1, 1, 1, 131, device=DEV).bfloat16()
    x, rows = wide[..., :128], wide[..., :128].clone(memory_format=torch.contiguous_format)
    pos = torch.tensor([5], device=DEV)
    for a, b in zip(qk_norm_rope(x, x, positions=pos), qk_norm_rope(rows, rows, positions=pos)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_one_gate_a_head_in_16_bits_has_one_rounding_of_its_gradient(dtype):
    """The gradient of a decay for each head is a sum over all tokens in fp32, rounded once to the gate's type, also where
    most of it cancels: the second row's gradient is nearly the first's negative."""
    x = _inputs(2, 600, 1, 8, 64, 64, "head", False, train=True, seed=33)
    for m in ("q", "k", "v", "do"):
        x[m][1] = x[m][0]
    x["do"][1] *= -1.0078125
    gate = x["g"].to(dtype)
    grads = []
    for g in (gate, gate.float()):
        g = g.detach().requires_grad_(True)
        o, _ = chunk_decay_linear_attention(x["q"], x["k"], x["v"], g, 0.1)
        grads.append(torch.autograd.grad(o, [g], [x["do"]])[0])
    assert grads[0].dtype == dtype and torch.equal(grads[0], grads[1].to(dtype))


def test_norm_rope_of_2_26_tokens():
    """A workgroup for every four tokens would be 2^32 threads, which no launch takes."""
    t = 2**26
    x = torch.randn(1, 4096, 1, 64, device=DEV).bfloat16().repeat(1, t // 4096, 1, 1)
    q, k = qk_norm_rope(x, x, rot_dim=64)
    for a, e in ((0, 300), (t // 2, t // 2 + 300), (t - 300, t)):
        want, _ = qk_norm_rope(x[:, a:e], x[:, a:e], rot_dim=64, positions=torch.arange(a, e, device=DEV))
        assert torch.equal(q[:, a:e], want) and torch.equal(k[:, a:e], want)
