"""GPU: values near the end of bf16's range, whose sums of weights times values pass fp32's before they are divided by the row's
sum: the results are averages of values and finite. Bounds: tests/window_ref.py."""
import pytest
import torch

from sorernn_amd import paged_attention, window_attention
from tests.test_gpu_paged import _cache
from tests.test_gpu_window import DEV, _inputs
from tests.window_ref import check, paged_attention as reference, window_attention as whole_reference

pytestmark = pytest.mark.gpu
MOST = torch.finfo(torch.bfloat16).max


@pytest.mark.parametrize("size", [1e35, 1e37, 3e37])
@pytest.mark.parametrize("t, d, win, sinks", [(300, 64, None, 0), (700, 128, 100, 3)])
def test_window(t, d, win, sinks, size):
    q, k, v, _ = _inputs(1, t, 2, 1, d, seed=1)
    v = (v.float() * size).bfloat16()
    check(window_attention(q, k, v, window=win, sinks=sinks), whole_reference(q, k, v, win, sinks, d**-0.5), "o")


def test_window_of_the_largest_value():
    q, k, v, _ = _inputs(1, 500, 2, 1, 64, seed=2)
    v.fill_(MOST)
    assert (window_attention(q, k, v) == MOST).all()
    v[:, :, :, 32:] = -MOST
    o = window_attention(q, k, v, window=90, sinks=2)
    assert (o[..., :32] == MOST).all() and (o[..., 32:] == -MOST).all()


@pytest.mark.parametrize("size", [1e35, 3e37])
@pytest.mark.parametrize("t, width", [(1, 8), (1, 60), (3, 60), (90, 20), (90, 100), (300, 60)])
def test_paged(t, width, size):
    n, hq, hkv, d, page = 2, 4, 2, 64, 16
    gen = torch.Generator(DEV).manual_seed(3)
    kc, vc, table = _cache(n, width * page, hkv, d, page, torch.bfloat16, gen)
    vc = (vc.float() * size).bfloat16()
    q = torch.randn(n, t, hq, d, generator=gen, device=DEV).bfloat16()
    lengths = torch.tensor([width * page, max(width * page - 37, t)], device=DEV)
    o = paged_attention(q, kc, vc, table, lengths)
    check(o, reference(q, kc, vc, table, lengths, None, 0, d**-0.5), "o")


@pytest.mark.parametrize("t, width", [(1, 8), (1, 60), (90, 20), (90, 100)])
def test_paged_of_the_largest_value(t, width):
    gen = torch.Generator(DEV).manual_seed(4)
    kc, vc, table = _cache(1, width * 16, 1, 128, 16, torch.bfloat16, gen)
    vc.fill_(MOST)
    q = torch.randn(1, t, 4, 128, generator=gen, device=DEV).bfloat16()
    o = paged_attention(q, kc, vc, table, torch.tensor([width * 16], device=DEV))
    assert (o == MOST).all()
