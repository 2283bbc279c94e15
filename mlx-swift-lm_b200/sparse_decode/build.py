"""Build libsparse_decode.so (sm_100a) in-tree with nvcc.

The library is compiled from mlx-swift-lm_b200/csrc: one object per storage
format (sd_inst.cu and, for the paged cache, sd_paged_inst.cu and sd_tree_inst.cu,
with SD_E/SD_BITS), the rotary and page-copy kernels (sd_rotary.cu), the plan
and row kernels of drafted tokens (sd_draft.cu) and their attention's tile
kernel (sd_tree_tile.cu), plus the C ABI (sd_api.cu, sd_pages.cu, sd_steps.cu).
The CUDA runtime is linked statically, so the .so only needs the driver at run
time.

`build(phase_timing=True)` makes a second library, libsparse_decode_phases.so,
compiled with -DSD_PHASE_TIMING: the decode kernel then writes per-phase
timestamps (sparse_decode.phase_profile reads them). The product library has
no stamps.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent.parent          # mlx-swift-lm_b200/
CSRC = PKG_DIR / "csrc"
BUILD = PKG_DIR / "_build"
LIB = PKG_DIR / "libsparse_decode.so"
LIB_PHASES = PKG_DIR / "libsparse_decode_phases.so"
INCLUDE = PKG_DIR.parent / "include"

NVCC = os.environ.get("NVCC", "nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
         f"-I{INCLUDE}", f"-I{CSRC}"]
FORMATS = [(e, b) for b in (0, 4, 8) for e in (0, 1, 2)]


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [
        INCLUDE / "sparse_decode.h"]


def _kernel_sources(name: str, skip: set) -> list[Path]:
    """What a kernel object depends on: its source and csrc's headers, less
    those of host code and of the other kernels."""
    return [CSRC / name] + [h for h in sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h"))
                            if h.name not in skip | {"sd_host.h", "sd_pages_host.h"}]


def _host_sources(name: str) -> list[Path]:
    return [CSRC / n for n in (name, "sd_format.h", "sd_params.h", "sd_kernels.h", "sd_host.h", "sd_paged.h",
                               "sd_pages_host.h", "sd_draft.h")] + [INCLUDE / "sparse_decode.h"]


def _stale(target: Path, sources: list[Path] | None = None) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(s.stat().st_mtime > t for s in (sources if sources is not None else _sources()))


def _run(cmd: list[str]) -> None:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"command failed ({r.returncode}): {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")


def build(force: bool = False, verbose: bool = False, phase_timing: bool = False) -> Path:
    """Compile every kernel object and link the shared library; returns its path."""
    lib = LIB_PHASES if phase_timing else LIB
    bdir = PKG_DIR / "_build_phases" if phase_timing else BUILD
    flags = FLAGS + (["-DSD_PHASE_TIMING"] if phase_timing else [])
    bdir.mkdir(exist_ok=True)
    # (object, source, extra flags, files it depends on)
    units = []
    tree = {"sd_tree.cuh", "sd_draft.h"}
    for e, b in FORMATS:
        fmt = [f"-DSD_E={e}", f"-DSD_BITS={b}"]
        units.append((f"sd_inst_e{e}_b{b}.o", "sd_inst.cu", fmt, _kernel_sources("sd_inst.cu", tree | {"sd_paged.cuh", "sd_paged.h"})))
        units.append((f"sd_paged_e{e}_b{b}.o", "sd_paged_inst.cu", fmt, _kernel_sources("sd_paged_inst.cu", tree | {"sd_decode.cuh"})))
        units.append((f"sd_tree_e{e}_b{b}.o", "sd_tree_inst.cu", fmt, _kernel_sources("sd_tree_inst.cu", {"sd_decode.cuh"})))
        if e == 2 or (e == 1 and b == 0):  # codes of bf16 pools alone
            units.append((f"sd_tree_tile_e{e}_b{b}.o", "sd_tree_tile.cu", fmt, _kernel_sources("sd_tree_tile.cu", {"sd_decode.cuh"})))
    units.append(("sd_rotary.o", "sd_rotary.cu", [],
                  _kernel_sources("sd_rotary.cu", tree | {"sd_decode.cuh", "sd_paged.cuh"})))
    units.append(("sd_draft.o", "sd_draft.cu", [],
                  _kernel_sources("sd_draft.cu", {"sd_tree.cuh", "sd_decode.cuh", "sd_paged.cuh"})))
    units += [(f"{n}.o", f"{n}.cu", [], _host_sources(f"{n}.cu")) for n in ("sd_api", "sd_pages", "sd_steps")]
    jobs = []
    for obj, src, extra, deps in units:
        if force or _stale(bdir / obj, deps):
            jobs.append([NVCC, *ARCH, *flags, *extra, "-c", str(CSRC / src), "-o", str(bdir / obj)])
    with cf.ThreadPoolExecutor(max_workers=max(2, os.cpu_count() or 2)) as ex:
        for f in cf.as_completed([ex.submit(_run, j) for j in jobs]):
            f.result()
            if verbose:
                print(".", end="", flush=True)
    objs = [str(bdir / obj) for obj, *_ in units]
    if not force and not jobs and not _stale(lib, [Path(o) for o in objs]):
        return lib
    tmp = lib.with_suffix(".so.tmp")
    _run([NVCC, *ARCH, "-shared", "-o", str(tmp), *objs, "-cudart=static"])
    tmp.replace(lib)
    if verbose:
        print(f" built {lib}")
    return lib


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, phase_timing="--phases" in sys.argv)
