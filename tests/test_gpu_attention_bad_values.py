"""GPU: infinities and NaN among the values anywhere in a sequence: who sees them has them, with their signs, and the call takes
about as long as another."""
import pytest
import torch

from sorernn_amd import paged_attention, window_attention
from tests.test_gpu_window import DEV, _inputs
from tests.test_gpu_window_bad_gradients import _ms
from tests.window_ref import check, paged_attention as paged_reference, window_attention as reference

pytestmark = pytest.mark.gpu
INF, NAN = torch.inf, torch.nan


@pytest.mark.parametrize("at", [0, 4000, 8000, 8100])
@pytest.mark.parametrize("win, sinks", [(None, 0), (1024, 4)])
def test_a_prompt_takes_no_longer(win, sinks, at):
    """A healthy call takes 0.11 to 0.35 ms; rows that see the infinity, or share a block with it, summed key by key took 3 to 25."""
    q, k, v, _ = _inputs(1, 8192, 16, 4, 128, seed=1)
    healthy = _ms(lambda: window_attention(q, k, v, window=win, sinks=sinks))
    v[0, at, :, 5] = INF
    bad = _ms(lambda: window_attention(q, k, v, window=win, sinks=sinks))
    print(f"{healthy:.2f} ms, {bad:.2f} ms")
    assert bad < 5 * healthy + 1, (healthy, bad)


@pytest.mark.parametrize("t", [1, 512])
@pytest.mark.parametrize("back", [3, 200, 5000])
def test_a_cache_takes_no_longer(t, back):
    gen = torch.Generator(DEV).manual_seed(2)
    kc, vc = (torch.randn(512, 4, 64, 128, generator=gen, device=DEV).bfloat16() for _ in range(2))
    table = torch.randperm(512, generator=gen, device=DEV).to(torch.int32).reshape(4, 128)
    lengths = torch.tensor([8192, 8192, 8000, 6000], device=DEV)
    q = torch.randn(4, t, 16, 128, generator=gen, device=DEV).bfloat16()
    healthy = _ms(lambda: paged_attention(q, kc, vc, table, lengths))
    place = 8192 - back
    vc[table[0, place // 64], :, place % 64, 9] = INF
    bad = _ms(lambda: paged_attention(q, kc, vc, table, lengths))
    print(f"{healthy:.2f} ms, {bad:.2f} ms")
    assert bad < 5 * healthy + 1, (healthy, bad)


# values at (token, column), and what a column is from a token on that sees them
SIGNS = [
    ([(40, 3, INF)], {3: INF}), ([(40, 3, -INF)], {3: -INF}), ([(40, 3, NAN)], {3: NAN}), ([(40, 3, INF), (41, 3, INF)], {3: INF}),
    ([(40, 3, INF), (77, 3, -INF)], {3: NAN}), ([(10, 0, -INF), (20, 63, INF), (30, 17, NAN)], {0: -INF, 63: INF, 17: NAN}),
    ([(5, c, INF if c % 2 else -INF) for c in range(64)], {c: INF if c % 2 else -INF for c in range(64)}),
]


def _check_signs(o, ref, seen_from, columns):
    for c, want in columns.items():
        col = o[..., c]
        assert torch.equal(col[:, seen_from:].nan_to_num(7, 8, 9), torch.full_like(col[:, seen_from:], want).nan_to_num(7, 8, 9)), c
    keep = [c for c in range(64) if c not in columns]
    for part, cols in ((slice(0, 5), slice(None)), (slice(0, None), keep)):
        check(o[:, part][..., cols], {m: y[:, part][..., cols] for m, y in ref.items()}, "o")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("spoiled, columns", SIGNS)
def test_signs(spoiled, columns, dtype):
    q, k, v, _ = _inputs(1, 300, 2, 1, 64, dtype, seed=3)
    ref = reference(q, k, v, None, 0, 0.125)
    for at, c, value in spoiled:
        v[0, at, 0, c] = value
    _check_signs(window_attention(q, k, v, scale=0.125), ref, 78, columns)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("t, width", [(290, 20), (290, 200), (16, 20), (16, 200)])
@pytest.mark.parametrize("spoiled, columns", SIGNS)
def test_signs_over_a_cache(spoiled, columns, t, width, dtype):
    """The last t of 300 tokens, tiles of 128 and 32 rows, one run and several."""
    gen = torch.Generator(DEV).manual_seed(4)
    kc, vc = (torch.randn(width + 1, 1, 16, 64, generator=gen, device=DEV).to(dtype) for _ in range(2))
    table = torch.arange(width, device=DEV, dtype=torch.int32)[None]
    q = torch.randn(1, t, 2, 64, generator=gen, device=DEV).to(dtype)
    lengths = torch.tensor([300], device=DEV)
    ref = paged_reference(q, kc, vc, table, lengths, None, 0, 0.125)
    for at, c, value in spoiled:
        vc[at // 16, 0, at % 16, c] = value
    o = paged_attention(q, kc, vc, table, lengths, scale=0.125)
    first = max(78 - (300 - t), 0)
    for c, want in columns.items():
        col = o[:, first:, :, c]
        assert torch.equal(col.nan_to_num(7, 8, 9), torch.full_like(col, want).nan_to_num(7, 8, 9)), c
    keep = [c for c in range(64) if c not in columns]
    if keep:
        check(o[..., keep], {m: y[..., keep] for m, y in ref.items()}, "o")
