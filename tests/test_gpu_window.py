"""GPU: attention with a window and sinks and its backward against 64 bits. Bounds: tests/window_ref.py."""
import pytest
import torch

from sorernn_amd import window, window_attention
from tests.window_ref import check, window_attention as reference

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _bounds(lens):
    return [0] + torch.tensor(lens).cumsum(0).tolist() if lens else None


def _inputs(b, t, hq, hkv, d, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator(DEV).manual_seed(seed)
    return [torch.randn(b, t, h, d, generator=gen, device=DEV).to(dtype) for h in (hq, hkv, hkv, hq)]  # q, k, v, do


CASES = [
    # B, T, HQ, HKV, D, window, sinks, lens
    (1, 1, 1, 1, 64, None, 0, None),
    (2, 63, 2, 1, 128, 16, 0, None),
    (1, 64, 4, 4, 64, 64, 1, None),
    (2, 65, 3, 1, 128, 1, 0, None),
    (1, 129, 2, 2, 64, 1, 3, None),
    (1, 200, 6, 2, 128, 50, 200, None),
    (1, 300, 2, 1, 64, 1000, 4, None),
    (3, 257, 5, 5, 64, 64, 64, None),
    (2, 513, 4, 2, 128, 100, 5, None),
    (1, 700, 2, 1, 128, None, 9, None),
    (1, 1100, 2, 1, 64, 70, 130, None),
    (2, 1500, 8, 8, 128, 200, 33, None),
    (1, 1000, 2, 1, 128, 64, 2, [1, 64, 65, 255, 256, 257, 1, 101]),
    (1, 1700, 4, 2, 64, 90, 4, [1300, 1, 399]),
    (1, 1900, 3, 3, 128, 5, 129, [900, 700, 300]),
    (1, 330, 3, 3, 64, None, 0, [1] * 130 + [200]),
]
IDS = [f"{c[0]}x{c[1]}-h{c[2]}.{c[3]}-{c[4]}-w{c[5]}.{c[6]}{'-docs' if c[7] else ''}" for c in CASES]


def _call(x, window, sinks, scale, bounds):
    cu = None if bounds is None else torch.tensor(bounds)
    return window_attention(*x, window=window, sinks=sinks, scale=scale, cu_seqlens=None if cu is None else cu.to(DEV),
                            cu_seqlens_cpu=cu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_forward(case, dtype):
    b, t, hq, hkv, d, win, sinks, lens = case
    *x, _ = _inputs(b, t, hq, hkv, d, dtype)
    o = _call(x, win, sinks, None, _bounds(lens))
    assert o.dtype == dtype and o.is_contiguous()
    check(o, reference(*x, win, sinks, d**-0.5, _bounds(lens)), "o")


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_backward(case):
    b, t, hq, hkv, d, win, sinks, lens = case
    *x, do = _inputs(b, t, hq, hkv, d, seed=1)
    leaves = [y.requires_grad_(True) for y in x]
    o = _call(leaves, win, sinks, 0.11, _bounds(lens))
    grads = torch.autograd.grad(o, leaves, do)
    with torch.no_grad():
        ref = reference(*x, win, sinks, 0.11, _bounds(lens), do)
    check(o.detach(), ref, "o")
    for name, g in zip(("dq", "dk", "dv"), grads):
        assert g.dtype == torch.bfloat16
        check(g, ref, name)
    again = torch.autograd.grad(_call(leaves, win, sinks, 0.11, _bounds(lens)), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))  # the same bits in every run
