"""Drafted tokens over the paged cache without a GPU: struct layout, shared
memory, and argument checks that answer before any launch."""
from __future__ import annotations

import ctypes
import subprocess

import pytest

import sparse_decode as sdp
from sparse_decode import SDPlan, paged

from test_abi import _c_layout
from test_paged import BAD_POOLS, _pages, native  # noqa: F401


def _status(native, rc):  # noqa: F811
    return sdp.STATUS[rc]


def test_struct_layout_matches_header():
    names = [f[0] for f in SDPlan._fields_]
    lay = _c_layout("sd_plan", names)
    assert lay["sizeof"] == ctypes.sizeof(SDPlan)
    for n in names:
        assert lay[n] == getattr(SDPlan, n).offset, n


def test_attend_ctas_fit_an_sm(tmp_path):
    """Two of the attend kernel, one of the tile kernel (with at most 4 KB of static shared memory), at every batch and format;
    the parts do not overlap."""
    src = tmp_path / "layout.cpp"
    src.write_text("""#include <cuda_runtime.h>
#include <cstdio>
#include "sd_draft.h"
using namespace sd;
int bad = 0;
template <int ESIZE, int BITS, int D> void all() {
  using F = PagedFmt<ESIZE, BITS, D>;
  for (int R = 4; R <= 16; R *= 2)
    for (int b = 1; b <= kPagedMaxBatch; ++b) {
      const PagedLayout l = tree_layout(b, R, D, ESIZE == 4 && BITS == 0, F::kStageBytes);
      const int pre = 4 * (2 * (b + 1) + 2 * (kTreeAttendThreads / 32) + 16);
      if (l.stages < 1 || l.q_off > l.buf_off || l.buf_off + 4 * kPagedWarps * paged_warp_floats(R, D) > l.prefix_off ||
          l.prefix_off + pre > l.bar_off || l.bar_off + 2 * 8 * l.stages + 1024 > l.bytes || 2 * (l.bytes + 1024) > 228 * 1024) ++bad;
    }
}
int main() {
  all<2, 0, 64>(); all<2, 0, 128>(); all<4, 0, 64>(); all<4, 0, 128>();
  all<2, 4, 64>(); all<2, 4, 128>(); all<4, 4, 64>(); all<4, 4, 128>();
  all<2, 8, 64>(); all<2, 8, 128>(); all<4, 8, 64>(); all<4, 8, 128>();
  for (int D = 64; D <= 128; D += 64)
    for (int x = 0; x < 6; ++x)
      for (int b = 1; b <= kPagedMaxBatch; ++b) {
        const int bits = x / 2 * 4, shared = x % 2;
        const TileLayout l = tree_tile_layout(b, D, bits, shared);
        const int raw = l.raw_stages * tree_raw_stage(D, bits);
        if (l.stages < kTreeTileLeast || l.stages > kTreeTileStages || ((bits || !shared) && l.stages % 4) || l.raw_stages % 2 || l.raw_stages > kTreeRawStages ||
            (bits && l.raw_stages < 2) || l.raw_off < (tree_tile_queries(D, bits, shared) * 128 + l.stages * kTreeTileTokens) * D * 2 ||
            l.raw_off % 128 || tree_raw_stage(D, bits) % 128 || l.prefix_off < l.raw_off + raw || l.bar_off % 8 ||
            l.prefix_off + 4 * (2 * (b + 1) + 2 * ((bits ? kTreeCodeThreads : kTreeTileThreads) / 32)) > l.bar_off ||
            l.bytes + 4096 > 227 * 1024) ++bad;
      }
  std::printf("%d", bad);
}
""")
    exe = tmp_path / "layout"
    csrc = sdp.LIB_PATH.parent / "csrc"
    subprocess.run(["g++", "-std=c++17", f"-I{csrc}", "-I/usr/local/cuda/include", str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout == "0"


def _plan(**kw):
    base = dict(lengths=256, added=256, tables=512, batch=2, table_width=3, page_size=16, n_rows=4, held=None, free_pages=None,
                taken=None, n_free=0, nodes=0, parents=None, parents_stride=0, first=256, ends=256, seq=256, positions=256,
                slots=None, places=None, masks=None)
    base.update(kw)
    return SDPlan(*base.values())


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), "SD_ERR_SHAPE"), (dict(batch=4097), "SD_ERR_SHAPE"), (dict(page_size=48), "SD_ERR_SHAPE"),
    (dict(table_width=-1), "SD_ERR_INVALID_ARG"), (dict(n_rows=-1), "SD_ERR_INVALID_ARG"), (dict(n_rows=1 << 30), "SD_ERR_SHAPE"),
    (dict(table_width=1 << 27), "SD_ERR_SHAPE"), (dict(lengths=None), "SD_ERR_INVALID_ARG"), (dict(added=None), "SD_ERR_INVALID_ARG"),
    (dict(tables=None), "SD_ERR_INVALID_ARG"), (dict(first=None), "SD_ERR_INVALID_ARG"), (dict(ends=None), "SD_ERR_INVALID_ARG"),
    (dict(seq=None), "SD_ERR_INVALID_ARG"), (dict(positions=None), "SD_ERR_INVALID_ARG"), (dict(held=256), "SD_ERR_INVALID_ARG"),
    (dict(held=256, taken=256, n_free=1), "SD_ERR_INVALID_ARG"), (dict(taken=256, free_pages=256), "SD_ERR_INVALID_ARG"),
    (dict(parents=256), "SD_ERR_SHAPE"), (dict(parents=256, nodes=65), "SD_ERR_SHAPE"), (dict(parents=256, nodes=4, parents_stride=-1), "SD_ERR_INVALID_ARG"),
    (dict(n_free=-1), "SD_ERR_INVALID_ARG"), (dict(lengths=258), "SD_ERR_INVALID_ARG"), (dict(slots=260), "SD_ERR_INVALID_ARG"),
    (dict(masks=260), "SD_ERR_INVALID_ARG"), (dict(places=257), "SD_ERR_INVALID_ARG")])
def test_plan_refusals(native, kw, status):  # noqa: F811
    assert _status(native, native.sd_paged_plan(_plan(**kw), None, None)) == status
    assert _status(native, native.sd_paged_plan(None, None, None)) == "SD_ERR_INVALID_ARG"


def test_plan_refuses_outputs_in_its_inputs(native):  # noqa: F811
    apart = dict(lengths=1 << 12, added=2 << 12, tables=3 << 12, held=4 << 12, free_pages=5 << 12, taken=6 << 12, n_free=5,
                 parents=7 << 12, nodes=4, parents_stride=6, first=8 << 12, ends=9 << 12, seq=10 << 12, positions=11 << 12,
                 slots=12 << 12, places=13 << 12, masks=14 << 12)
    sizes = dict(lengths=8, added=8, tables=24, held=8, free_pages=20, taken=4, parents=40)
    outs = dict(first=12, ends=8, seq=16, positions=16, slots=32, places=16, masks=32)
    for name, own in outs.items():
        for other, size in sizes.items():
            step = 8 if own == 32 else 4
            for at in (0, (size - 1) // step * step, -step):
                plan = _plan(**{**apart, name: apart[other] + at})
                assert _status(native, native.sd_paged_plan(plan, None, None)) == "SD_ERR_INVALID_ARG", (name, other, at)


def _tree(native, pages=None, layer=0, q=256, n_rows=4, batch=2, hq=8, tables=256, width=3, lengths=256, first=256,  # noqa: F811
          masks=None, places=None, scale=1.0, window=0, sinks=None, out=512, work=768, size=1 << 40, flags=None):
    return _status(native, native.sd_paged_tree_decode(pages or _pages(), layer, q, n_rows, batch, hq, tables, width, lengths, first,
                                                       masks, places, scale, window, sinks, out, work, size, flags, None))


@pytest.mark.parametrize("kw,status", [
    (dict(layer=2), "SD_ERR_INVALID_ARG"), (dict(layer=-1), "SD_ERR_INVALID_ARG"), (dict(batch=4097), "SD_ERR_SHAPE"),
    (dict(batch=-1), "SD_ERR_SHAPE"), (dict(n_rows=-1), "SD_ERR_INVALID_ARG"), (dict(hq=7), "SD_ERR_SHAPE"), (dict(hq=0), "SD_ERR_SHAPE"),
    (dict(hq=34), "SD_ERR_SHAPE"), (dict(q=None), "SD_ERR_INVALID_ARG"), (dict(q=264), "SD_ERR_INVALID_ARG"),
    (dict(out=520), "SD_ERR_INVALID_ARG"), (dict(work=None), "SD_ERR_INVALID_ARG"), (dict(work=772), "SD_ERR_INVALID_ARG"),
    (dict(tables=None), "SD_ERR_INVALID_ARG"), (dict(lengths=None), "SD_ERR_INVALID_ARG"), (dict(first=None), "SD_ERR_INVALID_ARG"),
    (dict(first=258), "SD_ERR_INVALID_ARG"), (dict(masks=260), "SD_ERR_INVALID_ARG"), (dict(places=258), "SD_ERR_INVALID_ARG"),
    (dict(sinks=258), "SD_ERR_INVALID_ARG"), (dict(flags=258), "SD_ERR_INVALID_ARG"), (dict(scale=float("inf")), "SD_ERR_INVALID_ARG"),
    (dict(window=-1), "SD_ERR_INVALID_ARG"), (dict(width=0), "SD_ERR_INVALID_ARG"), (dict(width=1 << 25), "SD_ERR_SHAPE"),
    (dict(batch=0), "SD_OK"), (dict(n_rows=0), "SD_OK")])
def test_tree_refusals(native, kw, status):  # noqa: F811
    assert _tree(native, **kw) == status


def _keep(native, pages=None, tables=4096, batch=2, width=3, ends=256, first=512, path=1024, path_width=4, kept=768, out=2048,  # noqa: F811
          flags=None):
    return _status(native, native.sd_paged_keep(pages or _pages(), tables, batch, width, ends, first, path, path_width, kept, out, flags, None))


@pytest.mark.parametrize("kw,status", [
    (dict(batch=4097), "SD_ERR_SHAPE"), (dict(batch=-1), "SD_ERR_SHAPE"), (dict(path_width=65), "SD_ERR_SHAPE"),
    (dict(path_width=-1), "SD_ERR_SHAPE"), (dict(width=0), "SD_ERR_INVALID_ARG"), (dict(width=1 << 25), "SD_ERR_SHAPE"),
    (dict(tables=None), "SD_ERR_INVALID_ARG"), (dict(ends=None), "SD_ERR_INVALID_ARG"), (dict(first=None), "SD_ERR_INVALID_ARG"),
    (dict(path=None), "SD_ERR_INVALID_ARG"), (dict(kept=None), "SD_ERR_INVALID_ARG"), (dict(out=None), "SD_ERR_INVALID_ARG"),
    (dict(ends=258), "SD_ERR_INVALID_ARG"), (dict(out=256), "SD_ERR_INVALID_ARG"), (dict(out=260), "SD_ERR_INVALID_ARG"),
    (dict(out=252), "SD_ERR_INVALID_ARG"), (dict(out=520), "SD_ERR_INVALID_ARG"), (dict(out=768), "SD_ERR_INVALID_ARG"),
    (dict(out=1052), "SD_ERR_INVALID_ARG"), (dict(out=4096), "SD_ERR_INVALID_ARG"), (dict(batch=0), "SD_OK")])
def test_keep_refusals(native, kw, status):  # noqa: F811
    assert _keep(native, **kw) == status


@pytest.mark.parametrize("kw,status", BAD_POOLS)
def test_every_call_refuses_a_bad_pool(native, kw, status):  # noqa: F811
    g = _pages(**kw)
    n = ctypes.c_int64()
    assert _status(native, native.sd_paged_tree_workspace(g, 1, 4, 8, ctypes.byref(n))) == status
    assert _tree(native, pages=g) == status
    assert _keep(native, pages=g) == status


def test_workspace_refusals(native):  # noqa: F811
    n = ctypes.c_int64(5)
    assert _status(native, native.sd_paged_tree_workspace(_pages(), 1, 4, 8, None)) == "SD_ERR_INVALID_ARG"
    assert _status(native, native.sd_paged_tree_workspace(_pages(), 0, 4, 8, ctypes.byref(n))) == "SD_OK" and n.value == 0
    assert _status(native, native.sd_paged_tree_workspace(_pages(), 4097, 4, 8, ctypes.byref(n))) == "SD_ERR_SHAPE"


def test_numbers_past_32_bits_are_refused_in_python():
    from sparse_decode import drafts
    assert drafts.MAX_NODES == 64
    with pytest.raises(ValueError):
        paged._count(1 << 31, "n_rows")
