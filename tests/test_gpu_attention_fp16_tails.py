"""GPU: fp16 attention whose rows give nearly all weight to one key, a sink, with a value of zero: the rest is the sum of many small
weights. Rounded to fp16 as they are, weights below 2^-14 of the largest would keep steps of 2^-24 and those below 2^-25 nothing.

The kernels' weights are at least 2^7 times larger against a row's sum, so that a term is off by half a step of fp16 of itself, or
by 2^-25 / 2^7 = 2^-32 of the sum. The rest of the bound is tests/window_ref.py's."""
import pytest
import torch

from sorernn_amd import paged_attention, window_attention
from tests.test_gpu_window import DEV
from tests.window_ref import check, half_step, one_head, seen

pytestmark = pytest.mark.gpu


def _inputs(t, length, d, gap, seed):
    """q [1,T,2,D], k, v [1,L,1,D] in fp16: key 0 scores `gap` above the others' mean at scale D^-0.5, the others spread by 1."""
    gen = torch.Generator(DEV).manual_seed(seed)
    q, k = (torch.randn(1, n, h, d, generator=gen, device=DEV) for n, h in ((t, 2), (length, 1)))
    q[..., 0] = 4
    k[..., 0] = 0
    k[:, 0] = 0
    k[:, 0, :, 0] = gap * d**0.5 / 4
    v = 1 + 0.5 * torch.randn(1, length, 1, d, generator=gen, device=DEV)
    v[:, 0] = 0
    return q.half(), k.half(), v.half()


def _reference(q, k, v, mask):
    d = q.shape[-1]
    out = {"o": torch.zeros(q.shape, dtype=torch.float64, device=DEV)}
    out["o_tol"] = torch.zeros_like(out["o"])
    for h in range(q.shape[2]):
        o, tol = one_head(q[0, :, h], k[0, :, 0], v[0, :, 0], mask, d**-0.5, half_step(torch.float16))
        out["o"][0, :, h], out["o_tol"][0, :, h] = o, tol + 2.0**-32 * (mask.double() @ v[0, :, 0].double().abs())
    return out


@pytest.mark.parametrize("gap", [9, 13, 16, 18])
@pytest.mark.parametrize("t, d, win, sinks", [(3000, 64, None, 0), (3000, 128, 700, 1)])
def test_window(t, d, win, sinks, gap):
    q, k, v = _inputs(t, t, d, gap, 1)
    at = torch.arange(t, device=DEV)
    check(window_attention(q, k, v, window=win, sinks=sinks), _reference(q, k, v, seen(at, at, win, sinks)), "o")


@pytest.mark.parametrize("gap", [9, 13, 16, 18])
@pytest.mark.parametrize("t, length", [(1, 250), (1, 8000), (40, 3000), (200, 6000)])
def test_paged(t, length, gap):
    q, k, v = _inputs(t, length, 64, gap, 2)
    pages = -(-length // 16)
    cache = []
    for x in (k, v):
        rows = torch.zeros(pages * 16, 64, device=DEV, dtype=torch.float16)
        rows[:length] = x[0, :, 0]
        cache.append(rows.view(pages, 16, 1, 64).transpose(1, 2).contiguous())
    table = torch.arange(pages, device=DEV, dtype=torch.int32)[None]
    o = paged_attention(q, *cache, table, torch.tensor([length], device=DEV))
    at = torch.arange(length, device=DEV)
    check(o, _reference(q, k, v, seen(at[length - t:], at, None, 0)), "o")
