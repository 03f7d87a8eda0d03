"""GPU: rows that see keys, but every score is -inf (an infinity in a key against the other sign in a query): their softmax is
0 / 0, NaN, and so is all that depends on it. Rows that see nothing stay zero. Bounds of the other rows: tests/window_ref.py."""
import pytest
import torch

from sorernn_amd import paged_attention, window_attention
from tests.test_gpu_window import DEV, _bounds, _inputs
from tests.test_gpu_window_more import _grads, _masked
from tests.window_ref import check, paged_attention as reference, window_attention as whole_reference

pytestmark = pytest.mark.gpu
COLUMN = 5  # keys hold +inf there, queries something negative


def _against(q):
    """Queries whose entry COLUMN is negative."""
    q = q.clone()
    q[..., COLUMN] = -1 - q[..., COLUMN].abs()
    return q


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("t, d, win, sinks, lens, at", [
    (1, 64, None, 0, None, [0]), (200, 128, None, 0, None, [0]), (200, 64, 1, 0, None, [0, 77, 199]),
    (300, 128, 2, 0, None, [70, 71]), (300, 64, 40, 3, [100, 1, 199], [0, 100, 101]), (150, 128, 1, 1, None, [0, 90]),
])
def test_window_forward(t, d, win, sinks, lens, at, dtype):
    q, k, v, _ = _inputs(1, t, 2, 1, d, dtype, seed=1)
    q = _against(q)
    k[0, at, 0, COLUMN] = torch.inf
    bounds = _bounds(lens)
    cu = None if bounds is None else torch.tensor(bounds, device=DEV)
    o = window_attention(q, k, v, window=win, sinks=sinks, cu_seqlens=cu)
    spans = [(0, t)] if bounds is None else list(zip(bounds[:-1], bounds[1:]))
    lost = torch.zeros(t, dtype=torch.bool, device=DEV)
    for s, e in spans:
        for i in range(s, e):
            seen = [j for j in range(s, i + 1) if win is None or i - j < win or j - s < sinks]
            lost[i] = all(j in at for j in seen)
    assert lost.any()
    assert o[:, lost].isnan().all() and o[:, ~lost].isfinite().all()


@pytest.mark.parametrize("t, d, win, sinks, at", [(1, 64, None, 0, 0), (200, 64, None, 0, 0), (300, 128, 1, 0, 130), (200, 128, 1, 2, 0)])
def test_window_gradients(t, d, win, sinks, at):
    q, k, v, do = _inputs(1, t, 2, 1, d, seed=2)
    q = _against(q)
    k[0, at, 0, COLUMN] = torch.inf
    got = dict(zip(("o", "dq", "dk", "dv"), _grads((q, k, v), do, window=win, sinks=sinks)))
    want = {"dk": 0, "dv": 0}
    for h in range(2):
        o, dq, dk, dv = _masked(q[0, :, h], k[0, :, 0], v[0, :, 0], do[0, :, h], win, sinks, d**-0.5)
        assert o[at].isnan().all()
        for name, y in (("o", o), ("dq", dq)):
            assert torch.equal(got[name][0, :, h].isfinite(), y.isfinite()), (name, h)
        want["dk"], want["dv"] = want["dk"] + dk, want["dv"] + dv
    for name in want:
        assert torch.equal(got[name][0, :, 0].isfinite(), want[name].isfinite()), name


def test_rows_of_no_document_stay_zero():
    from sorernn_amd import window

    q, k, v, do = _inputs(1, 300, 2, 1, 64, seed=3)
    q = _against(q)
    k[..., COLUMN] = torch.inf
    cu = torch.tensor([70, 130, 130, 250], device=DEV)
    o, kept = window.fwd_impl(q, k, v, cu, 40, 3, 0.125, 0, 3, True)
    grads = window.bwd_impl(q, k, v, o, kept, do, cu, 40, 3, 0.125, 0, 3)
    for y in (o, *grads):
        assert not y[:, :70].any() and not y[:, 250:].any() and y[:, 70:250].isnan().all()


# T new tokens a sequence, and table width in pages of 16: one run and several, tiles of 32 rows and of 128
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("t, width", [(1, 4), (1, 100), (3, 100), (90, 8), (90, 200), (300, 200)])
def test_paged(t, width, dtype):
    n, hq, hkv, d, page = 6, 4, 2, 64, 16
    most = width * page
    gen = torch.Generator(DEV).manual_seed(4)
    kc, vc = (torch.randn(n * width, hkv, page, d, generator=gen, device=DEV).to(dtype) for _ in range(2))
    table = torch.randperm(n * width, generator=gen, device=DEV).to(torch.int32).reshape(n, width)
    q = _against(torch.randn(n, t, hq, d, generator=gen, device=DEV).to(dtype))
    for m in (0, 2, 3, 4):  # the others' keys stay finite
        kc[table[m].long(), :, :, COLUMN] = torch.inf
    table[2] = -1                    # no page at all
    if width > 1:
        table[4, :-1] = -1           # only the last page
    lengths = torch.tensor([most, most, most, max(t // 2, 1), most, 0], device=DEV)
    o = paged_attention(q, kc, vc, table, lengths)
    place = lengths[:, None] - t + torch.arange(t, device=DEV)
    assert o[0].isnan().all()
    assert not o[2].any() and not o[5].any()
    assert o[3, place[3] >= 0].isnan().all() and not o[3, place[3] < 0].any()
    last = place[4] >= most - page
    assert o[4, last].isnan().all() and not o[4, ~last].any()
    one = slice(1, 2)
    check(o[one], reference(q[one], kc, vc, table[one], lengths[one], None, 0, d**-0.5), "o")


@pytest.mark.parametrize("t", [1, 40])
def test_paged_window_of_one(t):
    """Every row sees its own key alone: those against an infinity are lost, the others are their values."""
    gen = torch.Generator(DEV).manual_seed(5)
    kc, vc = (torch.randn(20, 1, 64, 128, generator=gen, device=DEV).bfloat16() for _ in range(2))
    table = torch.arange(20, device=DEV, dtype=torch.int32).reshape(1, 20)
    q = _against(torch.randn(1, t, 8, 128, generator=gen, device=DEV).bfloat16())
    length = 1200
    at = length - 1 - t // 2
    kc[at // 64, 0, at % 64, COLUMN] = torch.inf
    o = paged_attention(q, kc, vc, table, torch.tensor([length], device=DEV), window=1)
    values = vc[:, 0].flatten(0, 1)[length - t:length]
    for i in range(t):
        if length - t + i == at:
            assert o[0, i].isnan().all()
        else:
            assert torch.equal(o[0, i], values[i].expand(8, 128))


@pytest.mark.parametrize("base", [0, 700])
def test_paged_tree(base):
    """A drafted token that sees itself alone, with nothing in the cache before it, or with such keys alone before it."""
    gen = torch.Generator(DEV).manual_seed(6)
    kc, vc = (torch.randn(60, 2, 16, 64, generator=gen, device=DEV).bfloat16() for _ in range(2))
    table = torch.arange(60, device=DEV, dtype=torch.int32).reshape(1, 60)
    q = _against(torch.randn(1, 4, 4, 64, generator=gen, device=DEV).bfloat16())
    flat = kc.transpose(1, 2).reshape(960, 2, 64)  # a copy, by place
    flat[:base, :, COLUMN] = torch.inf
    flat[base + 1, :, COLUMN] = torch.inf
    kc = flat.reshape(60, 16, 2, 64).transpose(1, 2)
    # token 1 sees itself alone, token 2 itself, token 3 tokens 1 and 3, token 0 nothing drafted
    tree = torch.tensor([[0, 0b10, 0b100, 0b1010]], device=DEV)
    o = paged_attention(q, kc, vc, table, torch.tensor([base + 4], device=DEV), tree=tree)
    if base:
        assert o[0, 0].isnan().all()
    else:
        assert not o[0, 0].any()
    assert o[0, 1].isnan().all()
    values = vc.transpose(1, 2).reshape(960, 2, 64)
    for i in (2, 3):
        assert torch.equal(o[0, i], values[base + i].repeat_interleave(2, 0))


def test_whole_rows_are_unchanged():
    """Beside lost rows the others are those of the same inputs without the infinity, where they do not see it."""
    q, k, v, _ = _inputs(1, 400, 2, 1, 64, seed=7)
    q = _against(q)
    ref = whole_reference(q, k, v, 1, 0, 0.125)
    k[0, 200, 0, COLUMN] = torch.inf
    o = window_attention(q, k, v, window=1, scale=0.125)
    keep = torch.arange(400, device=DEV) != 200
    assert o[:, 200].isnan().all()
    check(o[:, keep], {m: y[:, keep] for m, y in ref.items()}, "o")
