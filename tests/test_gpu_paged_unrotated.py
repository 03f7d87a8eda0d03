"""GPU: the entries of appended rows that no rotation touches: without a norm they are the tokens' bits, and an infinity or NaN
among them changes no other."""
import pytest
import torch

from sorernn_amd import paged_kv_append
from tests.test_gpu_paged import DEV, U, _cache
from tests.linear_ref import check as check_rows, norm_rope

pytestmark = pytest.mark.gpu
SPECIAL = [torch.inf, -torch.inf, torch.nan, -0.0]


def _rows(dtype, d, rot, seed):
    """q, k, v of 70 tokens with special values in unrotated entries of q and k, one a row."""
    gen = torch.Generator(DEV).manual_seed(seed)
    q, k, v = (torch.randn(2, 35, h, d, generator=gen, device=DEV).to(dtype) for h in (4, 2, 2))
    for x in (q, k):
        flat = x.view(-1, d)
        at = torch.arange(flat.shape[0], device=DEV)
        flat[at, rot + at % (d - rot)] = torch.tensor(SPECIAL, device=DEV, dtype=dtype)[at % 4]
    return q, k, v


def _bits(x):
    return x.contiguous().view(torch.int16)


def _append(q, k, v, d, dtype, **kw):
    gen = torch.Generator(DEV).manual_seed(9)
    kc, vc, table = _cache(2, 64, 2, d, 16, dtype, gen)
    out = paged_kv_append(k, v, kc, vc, table, torch.tensor([60, 35], device=DEV), q=q, **kw)
    place = torch.stack([torch.arange(25, 60), torch.arange(35)]).to(DEV)
    at = table.long().gather(1, place // 16)
    return out, kc[at, :, place % 16], vc[at, :, place % 16], place


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d, rot", [(64, 0), (128, 0), (64, 16), (128, 32), (128, 64)])
def test_without_a_norm(d, rot, dtype):
    q, k, v = _rows(dtype, d, rot, 1)
    out, kn, vn, place = _append(q, k, v, d, dtype, rot_dim=rot)
    for got, x in ((out, q), (kn, k)):
        assert torch.equal(_bits(got[..., rot:]), _bits(x[..., rot:]))
        if rot:
            y = torch.where(x.isfinite(), x, 0).double()
            size = (y * y).mean(-1, keepdim=True).sqrt()
            ref = norm_rope(y / size, torch.ones(d, device=DEV), place, rot, 1e7, 0.0)
            check_rows(got[..., :rot], {"y": (ref["y"] * size)[..., :rot], "y_mag": (ref["y_mag"] * size)[..., :rot]}, "y", (d + 24) * U)
    assert torch.equal(_bits(vn), _bits(v))


@pytest.mark.parametrize("d, rot", [(64, 0), (128, 32)])
def test_with_a_norm(d, rot):
    """A row with an infinity has its other entries divided by one: zeros."""
    q, k, v = _rows(torch.bfloat16, d, rot, 2)
    w = torch.ones(d, device=DEV)
    out, kn, _, _ = _append(q, k, v, d, torch.bfloat16, rot_dim=rot, q_weight=w, k_weight=w)
    for got, x in ((out, q), (kn, k)):
        infinite = x.isinf().any(-1)
        row, was = got[infinite], x[infinite]
        assert row[was.isinf()].isnan().all() and not row[~was.isinf()].any()
        assert got[x.isnan().any(-1)].isnan().all() and got[x.isfinite().all(-1)].isfinite().all()
