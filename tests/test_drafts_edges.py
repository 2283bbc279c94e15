"""Drafted tokens without a GPU: trees on the host, the whole of the attend kernel's shared memory."""
from __future__ import annotations

import re
import subprocess

import sparse_decode as sdp

CSRC = sdp.LIB_PATH.parent / "csrc"


def test_lines_of_parents():
    from sparse_decode.paged import _lines
    assert _lines([]) == [] and _lines([-1, 0, 0, 1, -2, 4, -1]) == [1, 3, 5, 11, 0, 0, 64]
    assert _lines(list(range(-1, 63)))[-1] == (1 << 64) - 1


def test_attend_layout_has_room_for_all_that_the_kernel_places(tmp_path):
    """The numbers that the kernel lays out one behind the other, taken from its own lines, end before the barriers begin."""
    kernel = (CSRC / "sd_tree.cuh").read_text()
    kernel = kernel[kernel.index("tree_attend_kernel("):]
    assert "int* units = reinterpret_cast<int*>(sm + p.prefix_off);" in kernel
    line = next(x for x in kernel.splitlines() if "int *pairs = units" in x)
    chain = dict(re.findall(r"\*(\w+) = ([^,;]+)[,;]", line))
    assert list(chain) == ["pairs", "tmp", "low", "next"]
    counts = {int(i) for i in re.findall(r"next\[(\d)\]", (CSRC / "sd_tree.cuh").read_text())}
    src = tmp_path / "layout.cpp"
    src.write_text("""#include <cuda_runtime.h>
#include <cstdio>
#include "sd_draft.h"
using namespace sd;
int main() {
  int bad = 0;
  for (int b = 1; b <= kPagedMaxBatch; ++b) {
    struct { int B; } p{b};
    const int units = 0, pairs = %(pairs)s, tmp = %(tmp)s, low = %(low)s, next = %(next)s, end = next + %(counts)d;
    for (int D = 64; D <= 128; D += 64)
      for (int R = 4; R <= 16; R *= 2)
        for (int stage = 4096; stage <= 32768; stage *= 2)
          for (int f32 = 0; f32 < 2; ++f32) {
            const PagedLayout l = tree_layout(b, R, D, f32, stage);
            if (pairs != units + b + 1 || low - tmp < 2 * (kTreeAttendThreads / 32) || next - low < 16 || l.prefix_off + 4 * end > l.bar_off ||
                tree_attend_ints(b) != end) ++bad;
          }
  }
  std::printf("%%d", bad);
}
""" % {**chain, "counts": max(counts) + 1})
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", "-I/usr/local/cuda/include", str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout == "0"
