"""GPU: attention with a window and over a paged cache at the smallest scales, where all visible keys weigh the same."""
import pytest
import torch

from sorernn_amd import paged_attention, window_attention
from tests.test_gpu_window import DEV, _inputs
from tests.test_gpu_window_more import _grads
from tests.window_ref import check, window_attention as reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1e-30, 1e-38, 2e-45])
@pytest.mark.parametrize("win, sinks", [(None, 0), (50, 3)])
def test_window(win, sinks, scale):
    *x, do = _inputs(1, 300, 2, 1, 64, seed=21)
    o, _, _, dv = _grads(x, do, window=win, sinks=sinks, scale=scale)
    ref = reference(*x, win, sinks, scale, None, do)
    check(o, ref, "o")
    check(dv, ref, "dv")


@pytest.mark.parametrize("scale", [1e-38, 2e-45])
@pytest.mark.parametrize("t", [1, 3, 200])
def test_paged(t, scale):
    q, k, v, _ = _inputs(2, 1024, 4, 2, 128, seed=22)
    cache = [y.unflatten(1, (16, 64)).flatten(0, 1).transpose(1, 2).contiguous() for y in (k, v)]  # [pages, HKV, 64, D]
    table = torch.arange(32, device=DEV, dtype=torch.int32).reshape(2, 16)
    lengths = torch.tensor([1024, 1024], device=DEV)
    o = paged_attention(q[:, -t:], *cache, table, lengths, scale=scale)
    ref = reference(q, k, v, None, 0, scale)
    check(o, {m: y[:, -t:] for m, y in ref.items()}, "o")
