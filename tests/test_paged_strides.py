"""CPU: which strides of a paged cache the calls take. A dimension of one has whatever stride a view left it."""
import pytest
import torch

from sorernn_amd import paged_attention, paged_kv_append
from tests.test_window import launches  # noqa: F401  (the fixture)


def _view(shape, strides):
    room = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    return torch.zeros(room + 64).bfloat16().as_strided(shape, strides)


TABLE, LENGTHS = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([5])


@pytest.mark.parametrize("shape, strides, passed", [
    ((1, 2, 16, 64), (1, 1024, 64, 1), (0, 1024, 64)),
    ((3, 1, 16, 64), (1024, 3, 64, 1), (1024, 0, 64)),
    ((1, 1, 16, 64), (5, 7, 128, 1), (0, 0, 128)),
    ((3, 2, 16, 64), (2048, 1024, 64, 1), (2048, 1024, 64)),
    ((3, 2, 16, 64), (2048, 64, 128, 1), (2048, 64, 128)),
])
def test_strides_that_are_taken(launches, shape, strides, passed):  # noqa: F811
    kc, vc = _view(shape, strides), _view(shape, strides)
    hkv = shape[1]
    k = torch.zeros(1, 1, hkv, 64).bfloat16()
    paged_kv_append(k, k, kc, vc, TABLE, LENGTHS)
    paged_attention(torch.zeros(1, 1, 2 * hkv, 64).bfloat16(), kc, vc, TABLE, LENGTHS)
    append, attend = (args for _, args in launches)
    assert append[15] == kc.data_ptr() and append[16:19] == passed and append[19] == vc.data_ptr() and append[20:23] == passed
    assert attend[4] == kc.data_ptr() and attend[5:8] == passed and attend[8] == vc.data_ptr() and attend[9:12] == passed


@pytest.mark.parametrize("shape, strides", [
    ((3, 2, 16, 64), (2049, 1024, 64, 1)), ((3, 2, 16, 64), (2048, 1028, 64, 1)), ((1, 2, 16, 64), (1, 1025, 64, 1)),
    ((3, 1, 16, 64), (1025, 3, 64, 1)), ((1, 1, 16, 64), (8, 8, 65, 1)), ((1, 1, 16, 64), (8, 8, (1 << 23) + 8, 1)),
    ((3, 2, 16, 64), (2048, 1024, 1, 16)),
])
def test_strides_that_are_refused(launches, shape, strides):  # noqa: F811
    kc = _view(shape, strides)
    good = torch.zeros(shape).bfloat16()
    k = torch.zeros(1, 1, shape[1], 64).bfloat16()
    for caches in ((kc, good), (good, kc)):
        with pytest.raises(ValueError, match="contiguous and 16-byte aligned"):
            paged_kv_append(k, k, *caches, TABLE, LENGTHS)
        with pytest.raises(ValueError, match="contiguous and 16-byte aligned"):
            paged_attention(k, *caches, TABLE, LENGTHS)
    assert not launches
