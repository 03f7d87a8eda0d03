"""CPU: what the decay linear attention operators and the q/k norm with rotation refuse, their sizes and their route."""
import pytest
import torch

from sorernn_amd import _lib, linear, ops
from sorernn_amd import chunk_decay_linear_attention, fused_recurrent_decay_linear_attention, qk_norm_rope


@pytest.fixture
def launches(monkeypatch):
    """The checks of a call on CPU tensors, with the launches recorded."""
    calls = []
    monkeypatch.setattr(_lib, "call", lambda name, *a: calls.append(name))
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    for mod in (linear, ops):
        monkeypatch.setattr(mod, "_check_cuda", lambda name, *t: None)
    return calls


def _x(b=1, t=8, h=1, hv=2, kd=64, vd=64, dtype=torch.bfloat16):
    q = torch.randn(b, t, h, kd).to(dtype)
    return q, q.clone(), torch.randn(b, t, hv, vd).to(dtype), -torch.rand(b, t, hv)


def test_no_cpu_path():
    q, k, v, g = _x()
    for call in (lambda: chunk_decay_linear_attention(q, k, v, g), lambda: qk_norm_rope(q, k),
                 lambda: fused_recurrent_decay_linear_attention(q, k, v, g)):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("fn", [chunk_decay_linear_attention, fused_recurrent_decay_linear_attention])
def test_refusals_of_the_attention(fn, launches):
    q, k, v, g = _x()
    cases = [
        (ValueError, "expected", (q[0], k[0], v, g), {}),
        (ValueError, "expected", (q, k[:, :4], v, g), {}),
        (ValueError, "expected", (q, k, v[:, :4], g), {}),
        (ValueError, "multiple", (q.expand(1, 8, 3, 64), k.expand(1, 8, 3, 64), v, g), {}),
        (ValueError, "multiple", (q[:0], k[:0], v[:0], g[:0]), {}),
        (NotImplementedError, "head dims", (*(torch.randn(1, 8, 1, 32).bfloat16(),) * 3, None), {}),
        (NotImplementedError, "head dims", (q, k, torch.randn(1, 8, 2, 96).bfloat16(), g), {}),
        (ValueError, "share a dtype", (q, k, v.float(), g), {}),
        (TypeError, "dtype", (q.double(), k.double(), v.double(), g), {}),
        (TypeError, "dtype", (q, k, v, g.double()), {}),
        (ValueError, "g must be", (q, k, v, g[..., :1]), {}),
        (ValueError, "g must be", (q, k, v, torch.zeros(8)), {}),
        (ValueError, "initial_state", (q, k, v, g), {"initial_state": torch.zeros(1, 2, 64, 128)}),
        (ValueError, "cu_seqlens", (q, k, v, g), {"cu_seqlens": torch.tensor([0, 4, 4, 8])}),
        (ValueError, "cu_seqlens", (q, k, v, g), {"cu_seqlens": torch.tensor([0, 7])}),
        (ValueError, "cu_seqlens", (q, k, v, g), {"cu_seqlens": torch.tensor([0.0, 8.0])}),
        (ValueError, "B == 1", (*_x(2)[:3], None), {"cu_seqlens": torch.tensor([0, 8])}),
    ]
    for err, text, args, kw in cases:
        with pytest.raises(err, match=text):
            fn(*args, **kw)
    assert not launches


def test_refusals_of_gradients_and_in_place_states(launches):
    q, k, v, g = _x()
    qg = q.detach().requires_grad_(True)
    with pytest.raises(NotImplementedError, match="forward"):
        fused_recurrent_decay_linear_attention(qg, k, v, g)
    with pytest.raises(NotImplementedError, match="bf16"):
        chunk_decay_linear_attention(qg.float(), k.float(), v.float(), g)
    for h0 in (None, torch.zeros(1, 2, 64, 64).bfloat16(), torch.zeros(1, 2, 64, 128)[..., ::2]):
        with pytest.raises(ValueError, match="inplace_final_state"):
            fused_recurrent_decay_linear_attention(q, k, v, g, initial_state=h0, inplace_final_state=True)
    assert not launches


def test_refusals_of_the_norm(launches):
    q, k = torch.randn(2, 8, 4, 64).bfloat16(), torch.randn(2, 8, 2, 64).bfloat16()
    w = torch.ones(64)
    pos = torch.zeros(2, 8, dtype=torch.long)
    cases = [
        (ValueError, "expected", (q[0], k[0]), {}),
        (ValueError, "expected", (q, k[:, :4]), {}),
        (ValueError, "expected", (q, k[..., :32]), {}),
        (ValueError, "share a dtype", (q, k.float()), {}),
        (TypeError, "dtype", (q.double(), k.double()), {}),
        (ValueError, "no heads", (q[:, :, :0], k), {}),
        (ValueError, "weights", (q, k, w[:32]), {}),
        (ValueError, "weights", (q, k, w, torch.ones(1, 64)), {}),
        (NotImplementedError, "unsupported", (q[..., :32], k[..., :32]), {}),
        (NotImplementedError, "unsupported", (q, k), {"rot_dim": 24}),
        (NotImplementedError, "unsupported", (q, k), {"rot_dim": 128}),
        (NotImplementedError, "unsupported", (q, k), {"rot_dim": -16}),
        (ValueError, "positions", (q, k), {"positions": pos.float()}),
        (ValueError, "positions", (q, k), {"positions": pos[:1]}),
        (ValueError, "exclude", (q[:1], k[:1]), {"positions": pos[:1], "cu_seqlens": torch.tensor([0, 8])}),
        (ValueError, "B == 1", (q, k), {"cu_seqlens": torch.tensor([0, 8])}),
    ]
    for err, text, args, kw in cases:
        with pytest.raises(err, match=text):
            qk_norm_rope(*args, **kw)
    assert not launches


def test_calls_run_directly_and_one_gate_a_head_is_not_copied(launches):
    q, k, v, g = (x.requires_grad_(True) for x in _x(t=300))
    h0 = torch.zeros(1, 2, 64, 64, requires_grad=True)
    gh = torch.zeros(2, requires_grad=True)
    assert linear._gate_args(gh.expand(1, 300, 2)) == (_lib.DTYPE_F32, 0, 0, 1)
    o, s = chunk_decay_linear_attention(q, k, v, gh, initial_state=h0, output_final_state=True)
    grads = torch.autograd.grad([o, s], [q, k, v, gh, h0], [torch.ones_like(o), torch.ones_like(s)])
    assert [x.shape for x in grads] == [x.shape for x in (q, k, v, gh, h0)]
    with torch.no_grad():
        assert fused_recurrent_decay_linear_attention(q, k, v, g)[1] is None
    w = torch.ones(64, requires_grad=True)
    a, b = qk_norm_rope(q, k, w)
    torch.autograd.grad([a, b], [q, k, w], [torch.ones_like(a), torch.ones_like(b)])
    assert launches == ["gdn_decay_attn_fwd", "gdn_decay_attn_bwd", "gdn_decay_attn_recurrent_fwd", "gdn_qk_norm_rope_fwd",
                        "gdn_qk_norm_rope_bwd"]


def test_no_second_derivative(launches):
    q, k, v, g = (x.requires_grad_(True) for x in _x())
    o, _ = chunk_decay_linear_attention(q, k, v, g)
    (dq,) = torch.autograd.grad(o, [q], torch.ones_like(o), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.float().sum(), [k])


def test_a_state_overwritten_in_place_is_not_used_by_an_earlier_graph(launches):
    q, k, v, g = (x.requires_grad_(True) for x in _x())
    o, s = chunk_decay_linear_attention(q, k, v, g, output_final_state=True)
    with torch.no_grad():
        _, s2 = fused_recurrent_decay_linear_attention(q, k, v, g, initial_state=s, inplace_final_state=True)
        assert s2 is s
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad([o, s], [q], [torch.ones_like(o), torch.ones_like(s)])
    with torch.inference_mode():
        h0 = torch.zeros(1, 2, 64, 64)
        assert fused_recurrent_decay_linear_attention(q, k, v, g, initial_state=h0, inplace_final_state=True)[1] is h0


def test_sizes_match_the_library():
    lib = _lib.load()
    for b, t, hv, kd, vd, n, varlen in [(1, 1, 1, 64, 64, 1, 0), (4, 4096, 16, 128, 128, 4, 0), (1, 32768, 16, 128, 128, 8, 1),
                                        (1, 257, 1, 64, 128, 1, 0), (1, 257, 1, 64, 128, 257, 1), (1, 385, 2, 64, 64, 3, 1),
                                        (3, 385, 2, 64, 64, 3, 0), (2, 5000, 150, 64, 64, 2, 0), (2, 5000, 200, 64, 64, 2, 1), (64, 100, 16, 64, 64, 64, 0),
                                        (8, 300, 64, 128, 64, 8, 0), (1, 10**6, 1, 64, 64, 1, 0)]:
        assert linear.states_bytes(b, t, hv, kd, vd, bool(varlen)) == lib.gdn_decay_attn_states_size(
            b, t, hv, kd, vd, n, varlen)
    assert lib.gdn_decay_attn_states_size(0, 1, 1, 64, 64, 1, 0) == 0
    assert lib.gdn_decay_attn_bwd_workspace_size(1, 8, 2, 3, 64, 64, 1, 0) == 0
    assert lib.gdn_qk_norm_rope_bwd_workspace_size(1, 3, 64) == 3 * 2 * 64 * 4
    assert lib.gdn_qk_norm_rope_bwd_workspace_size(4, 4096, 128) == 512 * 2 * 128 * 4


def test_entry_points_check_their_arguments():
    """The C entry points refuse before any HIP call."""
    lib = _lib.load()
    P = 1 << 20  # an aligned address that is never read

    def fwd(q=P, k=P, v=P, o=P, cu=None, B=1, T=8, H=1, HV=1, K=64, V=64, N=1, gd=0, states=None, nb=0):
        return lib.gdn_decay_attn_fwd(q, k, v, None, None, o, None, cu, B, T, H, HV, K, V, N, gd, 0, 0, 0, 1.0, 0, states, nb,
                                      None)

    assert fwd(q=None) == _lib.GDN_ERR_INVALID
    assert fwd(q=P + 2) == _lib.GDN_ERR_INVALID and b"aligned" in lib.gdn_last_error()
    assert fwd(B=0) == _lib.GDN_ERR_INVALID
    assert fwd(H=2, HV=3) == _lib.GDN_ERR_INVALID
    assert fwd(N=2) == _lib.GDN_ERR_INVALID
    assert fwd(B=2, N=2, cu=P) == _lib.GDN_ERR_INVALID
    assert fwd(K=96) == _lib.GDN_ERR_UNSUPPORTED
    assert fwd(gd=3) == _lib.GDN_ERR_INVALID
    assert fwd(T=1000, HV=1) == _lib.GDN_ERR_INVALID and b"states" in lib.gdn_last_error()
    assert fwd(T=0) == _lib.GDN_OK
    bwd = [P, P, P, P, None, None, P, None, None, None, 1, 8, 1, 1, 64, 64, 1, 0, 0, 0, 0, 1.0, 0, P, P, P, P, None, None, 0, None]
    assert lib.gdn_decay_attn_bwd(*bwd) == _lib.GDN_ERR_INVALID and b"workspace" in lib.gdn_last_error()
    bwd[7] = P
    assert lib.gdn_decay_attn_bwd(*bwd) == _lib.GDN_ERR_INVALID and b"final_state" in lib.gdn_last_error()

    def rec(q=P, T=1, K=64, dt=1, h0=None, N=1):
        return lib.gdn_decay_attn_recurrent_fwd(q, P, P, None, h0, P, None, None, 1, T, 1, 1, K, 64, N, dt, 0, 0, 0, 0, 1.0, 0, None)

    assert rec(q=None) == _lib.GDN_ERR_INVALID and rec(N=2) == _lib.GDN_ERR_INVALID and rec(dt=5) == _lib.GDN_ERR_INVALID
    assert rec(h0=P + 4) == _lib.GDN_ERR_INVALID and rec(K=32) == _lib.GDN_ERR_UNSUPPORTED

    def rope(q=P, st=64, pos=None, cu=None, B=1, T=4, D=64, rot=16, theta=1e4, eps=1e-6, dt=1):
        return lib.gdn_qk_norm_rope_fwd(q, 0, st, 64, P, 0, 64, 64, None, None, pos, 0, 0, 0, P, P, cu, B, T, 1, 1, D, 1, dt, rot,
                                        theta, eps, 0, None)

    for kw in ({"q": None}, {"q": P + 8}, {"st": 65}, {"pos": P, "cu": P}, {"B": 2, "cu": P}, {"theta": 0.0}, {"eps": -1.0},
               {"theta": float("nan")}, {"eps": float("nan")}, {"dt": 7}):
        assert rope(**kw) == _lib.GDN_ERR_INVALID, kw
    for kw in ({"D": 96}, {"rot": 24}, {"rot": 80}):
        assert rope(**kw) == _lib.GDN_ERR_UNSUPPORTED, kw
    assert rope(T=0) == _lib.GDN_OK


@pytest.mark.parametrize("shape, pad", [((1, 1, 1), 131), ((1, 1, 3), 131), ((1, 4, 1), 131), ((2, 1, 1), 129)])
def test_padded_rows_are_copied_to_aligned_ones(shape, pad):
    """Also where the odd strides belong to dimensions of size 1, which a contiguous copy may keep."""
    x = torch.zeros(*shape, pad, dtype=torch.bfloat16)[..., :128]
    y, strides = linear._strided(x)
    assert torch.equal(x, y) and y.data_ptr() % 16 == 0 and strides[3] == 1
    assert all(st % 8 == 0 for st in strides[:3]) and all(n == 1 or st == s for n, st, s in zip(x.shape, strides, y.stride()))


def test_one_padded_row_reaches_the_kernels(launches, monkeypatch):
    """The C entry's own rule of alignment, for one token of one head."""
    def call(name, *a):
        launches.append(name)
        for at in (1, 2, 3, 5, 6, 7):
            assert a[at] % 8 == 0, (name, at, a[at])

    monkeypatch.setattr(_lib, "call", call)
    x = torch.zeros(1, 1, 1, 131, dtype=torch.bfloat16)[..., :128].requires_grad_(True)
    a, b = qk_norm_rope(x, x)
    torch.autograd.grad([a, b], [x], [torch.ones_like(a), torch.ones_like(b)])
    assert launches == ["gdn_qk_norm_rope_fwd", "gdn_qk_norm_rope_bwd"]


def test_launches_past_2_32_threads_are_refused():
    """A grid of more threads than 32 bits count is launched with what their number is modulo 2^32: most of the rows would
    silently stay as they were."""
    lib = _lib.load()
    P = 1 << 20
    for n, hv in ((2**18 + 3, 64), (2**24, 1), (2**18, 64)):
        assert lib.gdn_decay_attn_recurrent_fwd(P, P, P, None, None, P, None, None, n, 1, hv, hv, 64, 64, n, 1, 0, 0, 0, 0, 1.0, 0,
                                                None) == _lib.GDN_ERR_UNSUPPORTED, (n, hv)
    # dq and dk of the value heads that share a head: 1,024 elements a workgroup
    for t, h, hv in ((2**28, 1, 2), (2**26 + 5, 4, 8)):
        states = lib.gdn_decay_attn_states_size(1, t, hv, 64, 64, 1, 0)
        need = lib.gdn_decay_attn_bwd_workspace_size(1, t, h, hv, 64, 64, 1, 0)
        assert lib.gdn_decay_attn_bwd(P, P, P, None, None, None, P, None, P if states else None, None, 1, t, h, hv, 64, 64, 1, 0, 0,
                                      0, 0, 1.0, 0, P, P, P, None, None, P, need, None) == _lib.GDN_ERR_UNSUPPORTED, (t, h, hv)


def test_waves_share_a_token_up_to_a_workgroup_a_cu():
    """The norm's backward leaves a row of sums for each workgroup: one a token up to 256 tokens, then one for four."""
    size = _lib.load().gdn_qk_norm_rope_bwd_workspace_size
    assert [size(1, t, 64) // (2 * 64 * 4) for t in (1, 256, 257, 512, 2048, 4096)] == [1, 256, 65, 128, 512, 512]
