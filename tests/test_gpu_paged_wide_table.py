"""GPU: tables much wider than the sequences are long, as a server's are: what stands behind a sequence's last page does not
matter, whatever kernels and runs the width leads to. Bounds: tests/window_ref.py."""
import pytest
import torch

from sorernn_amd import paged_attention, paged_kv_append
from tests.test_gpu_paged import DEV, _cache
from tests.window_ref import check, gather, paged_attention as reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("behind", [-1, 0, 2**31 - 1])
@pytest.mark.parametrize("t, lengths, width", [
    (1, [33], 2048), (1, [700, 1, 16, 250], 512), (3, [700, 3], 1024), (40, [400, 41], 256), (130, [300, 131, 500], 600),
    (64, [1000], 4096),
])
def test_wide_tables(t, lengths, width, behind):
    gen = torch.Generator(DEV).manual_seed(1)
    n, longest = len(lengths), max(lengths)
    kc, vc, short = _cache(n, longest, 2, 64, 16, torch.bfloat16, gen)
    kc[0], vc[0] = torch.nan, torch.nan  # the page that a width's rest may name
    short = torch.where(short == 0, kc.shape[0] - 1, short) if not (short == kc.shape[0] - 1).any() else short
    for c in (kc, vc):
        c[short.unique().long()] = torch.randn(short.unique().numel(), 2, 16, 64, generator=gen, device=DEV).bfloat16()
    table = torch.full((n, width), behind, dtype=torch.int32, device=DEV)
    for m, length in enumerate(lengths):
        own = -(-length // 16)
        table[m, :own] = short[m, :own]
    lens = torch.tensor(lengths, device=DEV)
    q, k, v = (torch.randn(n, t, h, 64, generator=gen, device=DEV).bfloat16() for h in (8, 2, 2))
    q = paged_kv_append(k, v, kc, vc, table, lens, q=q, rot_dim=16)
    for win, sinks in ((None, 0), (100, 3)):
        o = paged_attention(q, kc, vc, table, lens, window=win, sinks=sinks)
        check(o, reference(q, kc, vc, table, lens, win, sinks, 0.125), "o")
    for m, length in enumerate(lengths):
        assert torch.equal(gather(vc, table[m], length)[length - t:], v[m])
