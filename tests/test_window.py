"""CPU: what attention with a window and sinks and the paged cache's calls refuse, their sizes and their route."""
import pytest
import torch

from sorernn_amd import _lib, linear, ops, paged, window
from sorernn_amd import paged_attention, paged_kv_append, window_attention


@pytest.fixture
def launches(monkeypatch):
    """The checks of a call on CPU tensors, with the launches recorded."""
    calls = []
    monkeypatch.setattr(_lib, "call", lambda name, *a: calls.append((name, a)))
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    for mod in (linear, ops, paged, window):
        monkeypatch.setattr(mod, "_check_cuda", lambda name, *t: None)
    return calls


def _x(b=1, t=8, hq=4, hkv=2, d=64, dtype=torch.bfloat16):
    return torch.randn(b, t, hq, d).to(dtype), *(torch.randn(b, t, hkv, d).to(dtype) for _ in range(2))


def _cache(n=1, width=4, hkv=2, size=16, d=64, dtype=torch.bfloat16):
    kc, vc = (torch.zeros(n * width + 1, hkv, size, d, dtype=dtype) for _ in range(2))
    return kc, vc, torch.arange(n * width, dtype=torch.int32).reshape(n, width), torch.full((n,), 20)


def test_no_cpu_path():
    q, k, v = _x()
    cache = _cache()
    for call in (lambda: window_attention(q, k, v), lambda: paged_kv_append(k, v, *cache), lambda: paged_attention(q, *cache)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_refusals_of_the_window(launches):
    q, k, v = _x()
    cases = [
        (ValueError, "expected", (q[0], k, v), {}),
        (ValueError, "expected", (q, k, v[:, :4]), {}),
        (ValueError, "expected", (q, k[:, :4], v[:, :4]), {}),
        (ValueError, "expected", (q, k[..., :32], v[..., :32]), {}),
        (ValueError, "multiple", (q[:, :, :3], k, v), {}),
        (ValueError, "multiple", (q[:, :, :0], k, v), {}),
        (ValueError, "multiple", (q, k[:, :, :0], v[:, :, :0]), {}),
        (ValueError, "multiple", (q[:0], k[:0], v[:0]), {}),
        (NotImplementedError, "head dim", (q[..., :32], k[..., :32], v[..., :32]), {}),
        (ValueError, "share a dtype", (q, k, v.half()), {}),
        (NotImplementedError, "bf16 or fp16", (q.float(), k.float(), v.float()), {}),
        (ValueError, "window", (q, k, v), {"window": 0}),
        (ValueError, "window", (q, k, v), {"window": -1}),
        (ValueError, "window", (q, k, v), {"window": 2.0}),
        (ValueError, "window", (q, k, v), {"window": True}),
        (ValueError, "sinks", (q, k, v), {"window": 4, "sinks": -1}),
        (ValueError, "cu_seqlens", (q, k, v), {"cu_seqlens": torch.tensor([0, 4, 4, 8])}),
        (ValueError, "cu_seqlens", (q, k, v), {"cu_seqlens": torch.tensor([0, 7])}),
        (ValueError, "B == 1", _x(2), {"cu_seqlens": torch.tensor([0, 8])}),
    ]
    for err, text, args, kw in cases:
        with pytest.raises(err, match=text):
            window_attention(*args, **kw)
    half = [y.half().requires_grad_(True) for y in (q, k, v)]
    with pytest.raises(NotImplementedError, match="bf16"):
        window_attention(*half)
    assert not launches
    with torch.no_grad():
        window_attention(*half)
    assert [name for name, _ in launches] == ["gdn_window_attn_fwd"]


def test_refusals_of_the_append(launches):
    q, k, v = _x()
    kc, vc, table, lengths = cache = _cache()
    w = torch.ones(64)
    cases = [
        (ValueError, "expected", (k[0], v[0], *cache), {}),
        (ValueError, "expected", (k, v[:, :4], *cache), {}),
        (ValueError, "expected", (k, v, *cache), {"q": q[:, :4]}),
        (ValueError, "expected", (k, v, *cache), {"q": q[:, :, :0]}),
        (ValueError, "share a dtype", (k, v.half(), *cache), {}),
        (ValueError, "share a dtype", (k, v, *cache), {"q": q.half()}),
        (ValueError, "share a dtype", (k, v, kc.half(), vc.half(), table, lengths), {}),
        (NotImplementedError, "head dim", (k[..., :32], v[..., :32], kc[..., :32], vc[..., :32], table, lengths), {}),
        (NotImplementedError, "bf16 or fp16", (k.float(), v.float(), kc.float(), vc.float(), table, lengths), {}),
        (ValueError, "caches must be", (k, v, kc[0], vc[0], table, lengths), {}),
        (ValueError, "caches must be", (k, v, kc, vc[:3], table, lengths), {}),
        (ValueError, "no pages", (k, v, kc[:0], vc[:0], table, lengths), {}),
        (ValueError, "heads", (k[:, :, :1], v[:, :, :1], *cache), {}),
        (NotImplementedError, "page size", (k, v, kc[:, :, :8], vc[:, :, :8], table, lengths), {}),
        (NotImplementedError, "page size", (k, v, *(torch.zeros(2, 2, 24, 64).bfloat16() for _ in range(2)), table, lengths), {}),
        (ValueError, "contiguous", (k, v, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, table, lengths), {}),
        (ValueError, "aligned", (k, v, kc, torch.zeros(vc.numel() + 1).bfloat16()[1:].view(vc.shape), table, lengths), {}),
        (ValueError, "page_table", (k, v, kc, vc, table.long(), lengths), {}),
        (ValueError, "page_table", (k, v, kc, vc, table[0], lengths), {}),
        (ValueError, "page_table", (k, v, kc, vc, table[:, :0], lengths), {}),
        (ValueError, "page_table", (k, v, kc, vc, table.repeat(2, 1), lengths), {}),
        (ValueError, "lengths", (k, v, kc, vc, table, lengths.float()), {}),
        (ValueError, "lengths", (k, v, kc, vc, table, lengths.repeat(2)), {}),
        (ValueError, "weights", (k, v, *cache), {"k_weight": w[:32]}),
        (ValueError, "without q", (k, v, *cache), {"q_weight": w}),
        (NotImplementedError, "rot_dim", (k, v, *cache), {"rot_dim": 24}),
        (NotImplementedError, "rot_dim", (k, v, *cache), {"rot_dim": 128}),
        (NotImplementedError, "rot_dim", (k, v, *cache), {"rot_dim": -16}),
        (ValueError, "positions", (k, v, *cache), {"positions": torch.zeros(1, 8)}),
        (ValueError, "positions", (k, v, *cache), {"positions": torch.zeros(2, 8, dtype=torch.long)}),
        (ValueError, "cu_seqlens", (k, v, *cache), {"cu_seqlens": torch.tensor([0, 7])}),
        (ValueError, "page_table", (k, v, *cache), {"cu_seqlens": torch.tensor([0, 4, 8])}),
        (NotImplementedError, "forward", (k.detach().requires_grad_(True), v, *cache), {}),
    ]
    for err, text, args, kw in cases:
        with pytest.raises(err, match=text):
            paged_kv_append(*args, **kw)
    assert not launches


def test_refusals_of_the_cached_attention(launches):
    q, k, v = _x()
    kc, vc, table, lengths = cache = _cache()
    tree = torch.zeros(1, 8, dtype=torch.int64)
    cases = [
        (ValueError, "expected", (q[0], *cache), {}),
        (ValueError, "multiple", (q[:, :, :3], *cache), {}),
        (ValueError, "no heads", (q[:, :, :0], *cache), {}),
        (ValueError, "no batch", (q[:0], *cache), {}),
        (ValueError, "share a dtype", (q.half(), *cache), {}),
        (NotImplementedError, "bf16 or fp16", (q.float(), kc.float(), vc.float(), table, lengths), {}),
        (ValueError, "caches must be", (torch.cat([q, q], 3), *cache), {}),
        (NotImplementedError, "page size", (q, kc[:, :, :1], vc[:, :, :1], table, lengths), {}),
        (ValueError, "page_table", (q, kc, vc, table.long(), lengths), {}),
        (ValueError, "lengths", (q, kc, vc, table, lengths[:0]), {}),
        (ValueError, "window", (q, *cache), {"window": 0}),
        (ValueError, "sinks", (q, *cache), {"sinks": -3}),
        (ValueError, "tree", (q, *cache), {"tree": tree.int()}),
        (ValueError, "tree", (q, *cache), {"tree": tree[:, :4]}),
        (NotImplementedError, "64 drafted", (q.repeat(1, 9, 1, 1), *cache), {"tree": tree.repeat(1, 9)}),
        (NotImplementedError, "64 drafted", (q.repeat(1, 9, 1, 1), kc, vc, table.repeat(2, 1), lengths.repeat(2)),
         {"tree": tree.repeat(1, 9), "cu_seqlens": torch.tensor([0, 65, 72])}),
        (ValueError, "cu_seqlens", (q, *cache), {"cu_seqlens": torch.tensor([0, 0, 8])}),
        (NotImplementedError, "forward", (q.detach().requires_grad_(True), *cache), {}),
    ]
    for err, text, args, kw in cases:
        with pytest.raises(err, match=text):
            paged_attention(*args, **kw)
    assert not launches
    paged_attention(q, *cache, tree=tree)
    paged_attention(q.repeat(1, 9, 1, 1), kc, vc, table.repeat(2, 1), lengths.repeat(2), tree=tree.repeat(1, 9),
                    cu_seqlens=torch.tensor([0, 64, 72]))
    assert [name for name, _ in launches] == ["gdn_paged_attn_fwd"] * 2


def test_views_are_read_in_place_and_others_copied(launches):
    """Strides that the kernels take go through as they are; a misaligned or too widely spaced tensor is copied."""
    d, hq, hkv = 64, 4, 2
    proj = torch.randn(2, 8, (hq + 2 * hkv) * d).bfloat16()
    q, k, v = (y.unflatten(-1, (-1, d)) for y in proj.split([hq * d, hkv * d, hkv * d], -1))
    window_attention(q, k, v)
    args = launches[-1][1]
    assert args[0] == q.data_ptr() and args[1:4] == q.stride()[:3] and args[4] == k.data_ptr() and args[8] == v.data_ptr()
    odd = torch.randn(2 * 8 * hkv * d + 1).bfloat16()[1:].view(2, 8, hkv, d)
    window_attention(q, odd, v)
    assert launches[-1][1][4] != odd.data_ptr() and launches[-1][1][5:8] == (8 * hkv * d, hkv * d, d)
    far = torch.zeros((1 << 23) + 72, dtype=torch.bfloat16).as_strided((1, 2, 1, 64), (0, (1 << 23) + 8, 0, 1))
    assert window._heads(far)[1] == (128, 64, 64, 1)


def test_training_runs_directly_and_has_no_second_derivative(launches):
    x = [y.requires_grad_(True) for y in _x(t=70)]
    o = window_attention(*x, window=5, sinks=2)
    grads = torch.autograd.grad(o, x, torch.ones_like(o), retain_graph=True)
    assert [g.shape for g in grads] == [y.shape for y in x]
    assert [name for name, _ in launches] == ["gdn_window_attn_fwd", "gdn_window_attn_bwd"]


def test_sizes_of_the_workspaces():
    lib = _lib.load()

    def align(n):
        return -(-n // 256) * 256

    size = lib.gdn_window_attn_bwd_workspace_size
    # delta alone: no sinks, no window, a window as long as the sequence
    assert size(2, 100, 4, 2, 64, 2, 10, 0, 0) == size(2, 100, 4, 2, 64, 2, 0, 5, 0) == size(2, 100, 4, 2, 64, 2, 99, 5, 0) == align(2 * 100 * 4 * 4)
    # a slot of 32 fp32 rows of dk and dv a kv head for each 256 far queries and each sequence
    assert size(2, 1000, 4, 2, 64, 2, 10, 5, 0) == align(2 * 1000 * 4 * 4) + (2 * 4 + 2) * 2 * 2 * 32 * 64 * 4
    # two tiles of sinks: pieces of 512, whole tiles of rows
    assert size(1, 1000, 4, 1, 128, 3, 10, 200, 1) == align(1000 * 4 * 4) + (1000 // 512 + 3 + 2 + 3) * 2 * 2 * 128 * 128 * 4
    assert size(0, 100, 4, 2, 64, 2, 10, 0, 0) == size(1, 100, 4, 2, 64, 2, -1, 0, 0) == 0
    size = lib.gdn_paged_attn_workspace_size
    # one token: 4 kv heads in 64 runs, of 32 rows with a maximum and a sum each
    assert size(1, 1, 16, 4, 128, 1, 64, 512, 0, 0, 0) == 4 * 64 * 32 * 130 * 4
    # as many tiles as there are CUs: one run
    assert size(64, 1, 16, 4, 128, 64, 16, 512, 0, 0, 0) == 0
    # a short cache makes no more runs than it has fours of blocks, one of 256 keys a single one
    assert size(1, 1, 16, 4, 128, 1, 64, 8, 0, 0, 0) == 4 * 5 * 32 * 130 * 4
    assert size(1, 1, 16, 4, 128, 1, 64, 4, 0, 0, 0) == 0
    # 244 rows a sequence: tiles of 32 while there is little to do, else of 128
    assert size(1, 61, 16, 4, 128, 1, 64, 16, 0, 0, 0) == 8 * 4 * 8 * 32 * 130 * 4
    assert size(8, 61, 16, 4, 128, 8, 64, 64, 0, 0, 0) == 16 * 4 * 8 * 128 * 130 * 4
    assert size(1, 1, 16, 4, 128, 1, 64, 1024, 300, 0, 0) == 4 * 3 * 32 * 130 * 4
    assert size(0, 1, 16, 4, 128, 1, 64, 512, 0, 0, 0) == size(1, 1, 15, 4, 128, 1, 64, 512, 0, 0, 0) == 0


def _call(name, **change):
    """An entry point's status for a valid call on made-up addresses with some arguments changed; nothing is launched, as every
    change makes it invalid."""
    a = 1 << 20
    orders = {
        "gdn_window_attn_fwd": "q qb qt qh k kb kt kh v vb vt vh o lse cu B T HQ HKV D N dtype window sinks scale flags stream",
        "gdn_window_attn_bwd": "q qb qt qh k kb kt kh v vb vt vh o lse do cu B T HQ HKV D N window sinks scale flags dq dk dv ws nbytes stream",
        "gdn_paged_append": "q qb qt qh k kb kt kh v vb vt vh qw kw qo kc kcp kch kct vc vcp vch vct table ts lengths li32 pos pb pt pi32 cu "
                            "B T HQ HKV D N pages size width dtype rot theta eps flags stream",
        "gdn_paged_attn_fwd": "q qb qt qh kc kcp kch kct vc vcp vch vct table ts lengths li32 tree tb tt o cu B T HQ HKV D N pages size width "
                              "dtype window sinks scale flags ws nbytes stream",
    }
    base = dict(q=a, k=a, v=a, o=a, lse=a, do=a, dq=a, dk=a, dv=a, ws=a, nbytes=1 << 30, cu=None, qb=4096, qt=512, qh=128, kb=4096, kt=512,
                kh=128, vb=4096, vt=512, vh=128, B=1, T=4, HQ=4, HKV=2, D=128, N=1, dtype=1, window=3, sinks=1, scale=0.1, flags=0,
                stream=None, qw=None, kw=None, qo=a, kc=a, kcp=4096, kch=2048, kct=128, vc=a, vcp=4096, vch=2048, vct=128, table=a,
                ts=4, lengths=a, li32=0, pos=None, pb=0, pt=0, pi32=0, pages=4, size=16, width=4, rot=32, theta=1e4, eps=1e-6,
                tree=None, tb=0, tt=0)
    base.update(change)
    return getattr(_lib.load(), name)(*(base[m] for m in orders[name].split()))


BOTH = [dict(B=0), dict(T=-1), dict(HKV=0), dict(N=0), dict(N=2), dict(cu=1 << 20, B=2, N=1), dict(D=96), dict(T=1 << 29), dict(HQ=70000)]
WINDOW = BOTH + [dict(HQ=3), dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                 dict(scale=float("inf")), dict(qt=513), dict(kh=-8), dict(kt=(1 << 23) + 8), dict(q=None), dict(v=(1 << 20) + 8)]
PAGED = BOTH + [dict(pages=0), dict(size=24), dict(size=8), dict(size=1 << 17), dict(width=0), dict(width=1 << 28), dict(dtype=0),
                dict(dtype=7), dict(kc=None), dict(table=None), dict(lengths=None), dict(kct=129), dict(vcp=-8), dict(pages=1 << 40)]


@pytest.mark.parametrize("name, changes", [
    ("gdn_window_attn_fwd", WINDOW + [dict(dtype=0), dict(o=None)]),
    ("gdn_window_attn_bwd", WINDOW + [dict(lse=None), dict(ws=None), dict(nbytes=8), dict(dq=None), dict(do=None)]),
    ("gdn_paged_append", PAGED + [dict(rot=24), dict(rot=144), dict(theta=0.0), dict(eps=-1.0), dict(k=None), dict(q=1 << 20, qo=None),
                                  dict(kt=4), dict(HQ=0)]),
    ("gdn_paged_attn_fwd", PAGED + [dict(HQ=3), dict(HQ=0), dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(o=None), dict(q=None),
                                    dict(kct=(1 << 23) + 8), dict(ws=None, width=64, window=0), dict(nbytes=100, width=64, window=0)]),
])
def test_entry_points_reject_bad_calls(name, changes):
    """Every check runs on the host before any launch (no GPU here: a call that passed them would report a HIP error)."""
    for change in changes:
        rc = _call(name, **change)
        assert rc in (_lib.GDN_ERR_INVALID, _lib.GDN_ERR_UNSUPPORTED), (change, rc, _lib.load().gdn_last_error())
        assert name.encode() in _lib.load().gdn_last_error()
    assert _call(name, T=0) == _lib.GDN_OK
