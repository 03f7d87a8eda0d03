"""CPU: a paged call's rows (tokens times heads of a group) have to fit the kernels' 32-bit row numbers; more are refused."""
import pytest

from sorernn_amd import _lib
from tests.test_window import _call


@pytest.mark.parametrize("change", [
    dict(T=1 << 27, HQ=4, HKV=1), dict(T=1 << 26, HQ=16, HKV=2), dict(T=(1 << 27) + 5, HQ=12, HKV=2), dict(T=1 << 27, HQ=64, HKV=1),
])
def test_too_many_rows_are_refused(change):
    """Tiles from row 2^29 on would be left out, and their outputs as they were."""
    assert change["T"] * change["HQ"] // change["HKV"] >= 1 << 29
    for more in (dict(), dict(cu=1 << 20)):
        # small enough strides and an 8-byte workspace: a call that passed this check would be refused by the next
        rc = _call("gdn_paged_attn_fwd", **change, **more, width=1 << 10, nbytes=8)
        assert rc == _lib.GDN_ERR_UNSUPPORTED and b"rows" in _lib.load().gdn_last_error()


def test_fewer_are_not():
    rc = _call("gdn_paged_attn_fwd", T=(1 << 27) - 1, HQ=4, HKV=1, o=None)
    assert rc == _lib.GDN_ERR_INVALID and b"rows" not in _lib.load().gdn_last_error().replace(b"rows not 16-byte", b"").replace(b"cache rows", b"")
