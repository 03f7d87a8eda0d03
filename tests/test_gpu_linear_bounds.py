"""GPU: documents' bounds as captured and compiled calls take them, unchecked: empty documents, tokens of none.

Error bounds: those of tests/test_gpu_linear.py.
"""
import pytest
import torch

from sorernn_amd import chunk_decay_linear_attention, fused_recurrent_decay_linear_attention, linear
from tests.linear_ref import check, decay_attention
from tests.test_gpu_linear import DEV, GATE, OUT, STATE, _block, _block_params, _inputs

pytestmark = pytest.mark.gpu

BOUNDS = [
    # tokens, bounds: sequences that stay whole (up to 384 tokens) and that are cut
    (300, [0, 200, 200]),                 # an empty document at the end, tokens behind it
    (300, [0, 1, 200, 200, 200, 200]),    # a call filled up to a fixed number of documents
    (300, [70, 70, 300]),                 # an empty one at the beginning, tokens before it
    (300, [0, 0, 130, 130, 131, 131]),
    (300, [0, 0, 0]),                     # no tokens at all
    (300, [300, 300, 300]),
    (700, [0, 300, 650, 650]),
    (700, [0, 650] + [650] * 200),
    (700, [130, 130, 390, 390, 390, 700]),
    (700, [0, 0, 0, 700, 700]),
    (700, [200, 200, 200]),
]
IDS = [f"{t}-{'.'.join(map(str, b[:6]))}" for t, b in BOUNDS]


def _run(t, bounds, h=1, hv=2, kd=64, vd=128, seed=21, states=True):
    """A forward and backward without checks, as a replay runs them."""
    n = len(bounds) - 1
    x = _inputs(1, t, h, hv, kd, vd, "token", True, [t // n] * (n - 1) + [t - t // n * (n - 1)], seed=seed, train=True)
    if not states:
        x["h0"] = x["dht"] = None
    cu = torch.tensor(bounds, device=DEV)
    args = [x[m] for m in ("q", "k", "v", "g", "h0")]
    o, final, kept = linear.attention_fwd_impl(*args, cu, 0.1, 0, n, True)
    grads = linear.attention_bwd_impl(*args, final, x["do"], x["dht"], kept, cu, 0.1, 0, n, True, True)
    torch.cuda.synchronize()
    return x, o, final, grads


@pytest.mark.parametrize("t, bounds", BOUNDS, ids=IDS)
def test_documents_among_empty_ones_and_loose_tokens(t, bounds):
    x, o, final, grads = _run(t, bounds)
    for n, (a, e) in enumerate(zip(bounds[:-1], bounds[1:])):
        if a == e:
            continue
        part = [x[m][:, a:e] for m in ("q", "k", "v", "g")]
        ref = decay_attention(*part, 0.1, x["h0"][n:n + 1], None, x["do"][:, a:e], x["dht"][n:n + 1])
        check(o[:, a:e], ref, "o", OUT)
        check(final[n:n + 1], ref, "state", STATE)
        for name, y in zip(("dq", "dk", "dv", "dg"), grads):
            check(y[:, a:e], ref, name, GATE if name == "dg" else OUT)
        check(grads[4][n:n + 1], ref, "dh0", STATE)


@pytest.fixture
def unwritten_is_nan():
    """Memory that nothing has written holds NaN."""
    torch.use_deterministic_algorithms(True, warn_only=True)
    yield
    torch.use_deterministic_algorithms(False)


@pytest.mark.parametrize("states", [True, False], ids=["states", "zeros"])
@pytest.mark.parametrize("t, bounds", BOUNDS, ids=IDS)
def test_states_of_empty_documents_go_through(t, bounds, states, unwritten_is_nan):
    """A document without tokens ends with its initial state, whose gradient is the final state's."""
    x, _, final, grads = _run(t, bounds, states=states)
    for n, (a, e) in enumerate(zip(bounds[:-1], bounds[1:])):
        if a == e:
            assert torch.equal(final[n], x["h0"][n] if states else torch.zeros_like(final[n])), n
            assert torch.equal(grads[4][n], x["dht"][n] if states else torch.zeros_like(final[n])), n
    assert torch.isfinite(final).all() and torch.isfinite(grads[4]).all()


def _loose(t, bounds):
    out = torch.ones(t, dtype=torch.bool, device=DEV)
    for a, e in zip(bounds[:-1], bounds[1:]):
        out[a:e] = False
    return out


@pytest.mark.parametrize("heads", [(1, 2), (2, 2)], ids=["shared", "own"])
@pytest.mark.parametrize("t, bounds", BOUNDS, ids=IDS)
def test_gradients_of_loose_tokens_are_zero(t, bounds, heads, unwritten_is_nan):
    _, _, _, grads = _run(t, bounds, *heads)
    loose = _loose(t, bounds)
    for name, y in zip(("dq", "dk", "dv", "dg"), grads):
        assert not y[:, loose].any() and torch.isfinite(y.float()).all(), name


def test_graph_of_a_training_step_with_loose_tokens(unwritten_is_nan):
    """Captured with whole bounds and replayed with padded ones, over memory full of NaN: the outputs of tokens in no
    document are zero, and the parameters' gradients those of the documents alone."""
    t, params = 700, _block_params(2)
    gen = torch.Generator(DEV).manual_seed(5)
    x, up = (torch.randn(1, t, 192, generator=gen, device=DEV).bfloat16() for _ in range(2))

    def step(x, up, cu, host):
        p = {n: w.detach().requires_grad_(True) for n, w in params.items()}  # leaves of this step's stream
        y, s = _block(x, p, cu, host)
        with torch.no_grad():  # the rows of the recurrent form too
            q = torch.ones(1, x.shape[1], 1, 64, device=DEV, dtype=x.dtype)
            o, _ = fused_recurrent_decay_linear_attention(q, q, q, cu_seqlens=cu, cu_seqlens_cpu=host)
        return [y, s, o, *torch.autograd.grad(y, list(p.values()), up)]

    host = torch.tensor([0, 100, 300, 700])
    cu, static = host.to(DEV), up.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(x, static, cu, host)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x, static, cu, host)
    for bounds in ([0, 200, 500, 500], [64, 64, 300, 650], [0, 100, 300, 700]):
        cu.copy_(torch.tensor(bounds))
        static.copy_(up)
        static[:, _loose(t, bounds)] = 0
        graph.replay()
        torch.cuda.synchronize()
        loose = _loose(t, bounds)
        for z in (outs[0], outs[2]):
            assert torch.isfinite(z).all() and not z[:, loose].any()
        a, e = bounds[0], bounds[-1]
        alone = sorted({b - a for b in bounds})
        want = step(x[:, a:e], up[:, a:e], torch.tensor(alone, device=DEV), torch.tensor(alone))
        for name, g, w in zip(params, outs[3:], want[3:]):
            assert torch.isfinite(g).all(), name
            if name in ("w", "wo"):  # a few roundings to bf16 on the way, each of half a step at most
                assert (g.double() - w.double()).norm() <= 8 * 2.0**-8 * w.double().norm(), name


def test_compiled_call_with_loose_tokens(unwritten_is_nan):
    """A compiled function does not read the bounds: padded ones give what a replay gives."""
    def f(q, k, v, g, h0, cu):
        return chunk_decay_linear_attention(q, k, v, g, 0.1, h0, True, cu)

    torch._dynamo.reset()
    compiled = torch.compile(f, fullgraph=True, backend="aot_eager")
    t, bounds = 700, [64, 64, 300, 650, 650]
    x = _inputs(1, t, 1, 2, 64, 128, "token", True, [100, 100, 100, 400], seed=23, train=True)
    leaves = [x[m].requires_grad_(True) for m in ("q", "k", "v", "g", "h0")]
    o, s = compiled(*leaves, torch.tensor(bounds, device=DEV))
    grads = torch.autograd.grad([o, s], leaves, [x["do"], x["dht"]])
    loose = _loose(t, bounds)
    for y in (o, *grads[:4]):
        assert torch.isfinite(y).all() and not y[:, loose].any()
    with torch.no_grad():
        for n in (0, 3):
            assert torch.equal(s[n], x["h0"][n]) and torch.equal(grads[4][n], x["dht"][n])
        for n, (a, e) in ((1, (64, 300)), (2, (300, 650))):
            part = [x[m][:, a:e] for m in ("q", "k", "v", "g")]
            ref = decay_attention(*part, 0.1, x["h0"][n:n + 1], None, x["do"][:, a:e], x["dht"][n:n + 1])
            check(o[:, a:e], ref, "o", OUT)
            for name, y in zip(("dq", "dk", "dv", "dg"), grads):
                check(y[:, a:e], ref, name, GATE if name == "dg" else OUT)
    torch._dynamo.reset()
