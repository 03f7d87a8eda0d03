"""GPU: gradients where rows see few keys, so that do.v - do.o is small against do.o: the relative error over all entries.

Roundings of half a step h = 2^-8 at most, uniform in it: rms h / sqrt(3) of a value where mantissas are evenly spread, 0.7 of
that on average. A gradient's are p's (in o, which do.o takes over), ds's and its own: sqrt(3) times one, 2 times with what
their sums' signs leave. With o's rounding among them the errors here were 2.5 times one rounding's."""
import pytest
import torch

from tests.test_gpu_window import DEV, _bounds, _call, _inputs
from tests.window_ref import window_attention as reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t, hq, hkv, d, win, sinks, lens", [
    (2000, 4, 2, 128, 2, 0, None), (2000, 4, 2, 64, 3, 0, None), (1000, 8, 1, 128, 2, 1, None), (600, 2, 2, 64, None, 0, [3] * 200),
])
def test_errors_are_those_of_the_roundings(t, hq, hkv, d, win, sinks, lens):
    *x, do = _inputs(1, t, hq, hkv, d, seed=31)
    leaves = [y.requires_grad_(True) for y in x]
    grads = torch.autograd.grad(_call(leaves, win, sinks, None, _bounds(lens)), leaves, do)
    with torch.no_grad():
        ref = reference(*x, win, sinks, d**-0.5, _bounds(lens), do)
    for name, g in zip(("dq", "dk", "dv"), grads):
        want = ref[name]
        one = (want.to(torch.bfloat16).double() - want).norm() / want.norm()
        error = (g.double() - want).norm() / want.norm()
        print(name, float(one), float(error / one))
        assert error <= 2 * one, (name, float(error / one))
