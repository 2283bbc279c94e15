"""The paged cache's calls at the ends of their ranges, without a GPU: every
answer here comes before a launch."""
from __future__ import annotations

import pytest

import sparse_decode as sdp
from sparse_decode import paged

from test_paged import _decode, _pages, _rotary, native  # noqa: F401


# -- counts ---------------------------------------------------------------------

@pytest.mark.parametrize("batch,tokens", [(65536, 65536), (1 << 16, 1 << 15), (1, (1 << 31) - 1), (1, (1 << 31) - 64),
                                          (2, (1 << 30) - 32), ((1 << 31) - 1, (1 << 31) - 1)])
def test_rotary_refuses_more_tokens_than_an_index_holds(native, batch, tokens):  # noqa: F811
    """One head of two elements: fewer warps than 2^31, but more tokens."""
    rows = paged.SDRows(256, 2 * tokens, 2, 2)
    assert _rotary(native, dict(rot_dim=2), dim=2, batch=batch, tokens=tokens, hq=1, q=rows, qo=rows, hkv=0, k=None,
                   ko=None) == "SD_ERR_SHAPE"


def test_append_refuses_more_tokens_than_an_index_holds(native):  # noqa: F811
    rows = paged.SDRows(256, 0, 64, 64)
    g = _pages(n_kv_heads=1, head_dim=64)
    for n in ((1 << 31) - 1, (1 << 31) - 64):
        rc = native.sd_paged_append(g, 0, n, rows, rows, 256, 1, 1, 256, None, None, 0, None, None, None, None)
        assert sdp.STATUS[rc] == "SD_ERR_SHAPE"


@pytest.mark.parametrize("kv,G", [(8192, 16), (65537, 1), (1 << 21, 16)])
def test_decode_refuses_heads_past_its_32_bit_rows(native, kv, G):  # noqa: F811
    """The join of the segments indexes a sequence's output by head * D in 32 bits."""
    import ctypes
    g = _pages(n_kv_heads=kv, page_size=16, n_pages=1)
    assert _decode(native, g=g, heads=kv * G, batch=1, width=1) == "SD_ERR_SHAPE"
    n = ctypes.c_int64()
    assert sdp.STATUS[native.sd_paged_workspace(g, 1, kv * G, ctypes.byref(n))] == "SD_ERR_SHAPE"
