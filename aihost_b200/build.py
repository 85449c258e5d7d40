"""Build libaihost_attn.so (the C-ABI attention library) in-tree with nvcc for sm_100a.

Beside it goes the Python module _kv8 (host C++ over the library and torch's headers).

Usage: python -m aihost_b200.build [--force] [--verbose]
The library is written next to this file; a build is skipped when it is newer than every source.
"""
from __future__ import annotations

import argparse
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libaihost_attn.so"
MODULE = PKG / "_kv8.so"
OBJ = PKG / "_build"  # one object file per source (ignored by git)
SOURCES = ["api.cu", "rope_append.cu", "decode.cu", "prefill_sm100.cu", "noalloc.cu", "decode_mma.cu", "dist.cu",
           "matmul_sm100.cu", "kv8_api.cu", "kv8_pages.cu", "kv8_append.cu", "kv8_attn.cu",
           "kv8_prefill_sm100.cu"]
HEADERS = ["common.cuh", "kernels.h", "rows.cuh"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    return "nvcc"


def _deps(src: str) -> list[Path]:
    own = ["ctx.h"] if src == "api.cu" or src == "kv8_api.cu" else []
    own += ["kv8.h", "kv8_tile.cuh"] if src.startswith("kv8_") or src == "api.cu" else []
    return [CSRC / h for h in [src] + HEADERS + own] + [ROOT / "include" / "aihost_attn.h", Path(__file__)]


def _stale(out: Path, deps: list[Path]) -> bool:
    return not out.exists() or any(p.stat().st_mtime >= out.stat().st_mtime for p in deps)


def needs_build() -> bool:
    return any(_stale(LIB, _deps(s)) for s in SOURCES) or _module_stale()


def _module_stale() -> bool:
    return _stale(MODULE, [CSRC / "kv8_py.cpp", ROOT / "include" / "aihost_attn.h", Path(__file__)])


def _build_module(verbose: bool) -> None:
    """_kv8.so, which finds the library and torch's own at run time (torch is imported first)."""
    import sysconfig

    import torch

    base = Path(torch.__file__).resolve().parent
    tmp = f"{MODULE}.{os.getpid()}.tmp"
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          f"-I{base / 'include'}", f"-I{base / 'include/torch/csrc/api/include'}",
          f"-I{sysconfig.get_paths()['include']}", f"-I{Path(nvcc_path()).resolve().parent.parent / 'include'}",
          "-o", tmp, str(CSRC / "kv8_py.cpp"), f"-L{base / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python",
          f"-L{PKG}", f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN"], MODULE.name, verbose)
    os.replace(tmp, MODULE)


def _run(cmd: list[str], what: str, verbose: bool) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({res.returncode}) building {what}")


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile what changed, one object per source and all of them at once, then link."""
    if not force and not needs_build():
        return LIB
    OBJ.mkdir(exist_ok=True)
    common = [nvcc_path(), "-O3", "-std=c++17", "-lineinfo", "-gencode", "arch=compute_100a,code=sm_100a",
              "-Xcompiler", "-fPIC", "-Xptxas", "-v" if verbose else "-O3"]

    def compile_one(src: str) -> None:
        obj = OBJ / (src + ".o")
        if not force and not _stale(obj, _deps(src)):
            return
        tmp = f"{obj}.{os.getpid()}.tmp.o"
        _run(common + ["-c", "-o", tmp, str(CSRC / src)], src, verbose)
        os.replace(tmp, obj)

    if force or any(_stale(LIB, _deps(s)) for s in SOURCES):
        with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
            list(pool.map(compile_one, SOURCES))
        _run(common + ["-shared", "-Xlinker", f"-soname={LIB.name}", "-o", str(LIB) + ".tmp"] +
             [str(OBJ / (s + ".o")) for s in SOURCES] + ["-ldl"], LIB.name, verbose)
        os.replace(str(LIB) + ".tmp", LIB)
    if force or _module_stale():
        _build_module(verbose)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
