"""The paged cache's calls at the ends of their ranges, without a GPU: every
answer here comes before a launch."""
from __future__ import annotations

import subprocess

import pytest

import sparse_decode as sdp
from sparse_decode import paged

from test_paged import _decode, _pages, _rotary, native  # noqa: F401


# -- residency ------------------------------------------------------------------

def test_two_decode_ctas_fit_an_sm(tmp_path):
    """For every format, head count and batch, from the layout that the launch uses: an SM has 228 KB and keeps 1 KB of
    it per CTA. Static shared memory would come on top; the decode kernel has none."""
    src = tmp_path / "layout.cpp"
    src.write_text("""#include <cuda_runtime.h>
#include <cstdio>
#include "sd_paged.h"
using namespace sd;
int bad = 0, full = 0;
template <int ESIZE, int BITS, int D> void all() {
  using F = PagedFmt<ESIZE, BITS, D>;
  for (int G = 1; G <= 16; ++G)
    for (int b = 1; b <= kPagedMaxBatch; ++b) {
      const PagedLayout l = paged_layout(b, G, D, ESIZE == 4 && BITS == 0, F::kStageBytes);
      const int parts = l.q_off <= l.buf_off && l.buf_off + 4 * kPagedWarps * paged_warp_floats(G, D) <= l.prefix_off &&
                        l.prefix_off + 4 * (b < 32 ? 160 : b + 1 + 5) <= l.bar_off && l.bar_off + 2 * 8 * l.stages + 1024 <= l.bytes;
      if (l.stages < 1 || !parts || 2 * (l.bytes + 1024) > 228 * 1024) ++bad;
      full += l.bytes == kPagedSmem;
    }
}
int main() {
  all<2, 0, 64>(); all<2, 0, 128>(); all<4, 0, 64>(); all<4, 0, 128>();
  all<2, 4, 64>(); all<2, 4, 128>(); all<4, 4, 64>(); all<4, 4, 128>();
  all<2, 8, 64>(); all<2, 8, 128>(); all<4, 8, 64>(); all<4, 8, 128>();
  std::printf("%d %d", bad, full);
}
""")
    exe = tmp_path / "layout"
    csrc = sdp.LIB_PATH.parent / "csrc"
    subprocess.run(["g++", "-std=c++17", f"-I{csrc}", "-I/usr/local/cuda/include", str(src), "-o", str(exe)], check=True)
    bad, full = map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    assert bad == 0
    assert full > 0  # some calls fill their share to the last byte: nothing may be added to it


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


def test_rows_of_more_tokens_than_32_bits_are_refused():
    """A ctypes argument keeps the low 32 bits of a larger number, so the calls refuse it first."""
    import torch
    x = torch.zeros(2)
    for n in ((1 << 32) + 5, 1 << 31):
        with pytest.raises(ValueError, match="2\\^31"):
            paged._rows(x.as_strided((n, 1, 2), (0, 0, 1)), "q", x.dtype, -1, 2)
        with pytest.raises(ValueError, match="2\\^31"):
            paged._rows(x.as_strided((n, 1, 1, 2), (0, 0, 0, 1)), "q", x.dtype, -1, 2)
    assert paged._rows(x.as_strided(((1 << 31) - 1, 1, 2), (0, 0, 1)), "q", x.dtype, -1, 2)[2] == (1 << 31) - 1


@pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 16, 1 << 62, -(1 << 32) + 5])
def test_counts_past_32_bits_are_refused(n):
    with pytest.raises(ValueError, match="window"):
        paged._count(n, "window")


@pytest.mark.parametrize("n", [0, -1, 7, (1 << 31) - 1, -(1 << 31)])
def test_counts_of_32_bits_pass(n):
    assert paged._count(n, "window") == n


@pytest.mark.gpu
def test_calls_refuse_layers_and_windows_past_32_bits(cuda):
    import torch
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    p, i32 = sdp.KVPages(z(2, 1, 16, 64), z(2, 1, 16, 64)), torch.int32
    q, k, t, n = z(1, 4, 64), z(1, 1, 64), z(1, 1, dt=i32), torch.ones(1, dtype=i32, device="cuda")
    far = 1 << 32
    for bad in (lambda: sdp.paged_decode(q, p, t, n, window=far + 16), lambda: sdp.paged_decode(q, p, t, n, layer=far),
                lambda: sdp.paged_append(p, k, k, t, n - 1, layer=far)):
        with pytest.raises(ValueError):
            bad()


# -- the router -------------------------------------------------------------------

def test_router_looks_up_nothing_per_call(monkeypatch):
    """A layer's call takes microseconds: the router's import of the paged layers is made once, not in each of them."""
    import sys

    import torch
    monkeypatch.setitem(sys.modules, "sparse_decode.paged", None)  # an import now fails
    x = torch.randn(1, 2, 3, 64)
    assert sdp.attention_with_cache_update(x, x, x, None, 0.1).shape == x.shape
    with pytest.raises(TypeError):
        sdp.attention_with_cache_update(x, x, x, object(), 0.1)
