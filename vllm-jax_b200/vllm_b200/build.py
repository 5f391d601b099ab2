"""Build libvjattn.so (the sm_100a kernels + C ABI) in-tree with nvcc, and
_torch_calls.so (argument checks and launches of the shortest calls, against
torch's C++ headers) with g++.

The shared libraries are written next to this file so that they travel with the
source tree; nothing is installed into site-packages. Usage:

    python -m vllm_b200.build            # incremental
    python -m vllm_b200.build --force    # rebuild everything
    python -m vllm_b200.build --ptxas-v  # print registers / spills per kernel
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

from . import _native

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR.parent / "csrc"
INCLUDE = PKG_DIR.parent.parent / "include"
BUILD_DIR = PKG_DIR.parent / "_build"
LIB_NAME = "libvjattn.so"
LIB_PATH = PKG_DIR / LIB_NAME
CALLS_SRC = CSRC / "torch_calls.cpp"
CALLS_PATH = PKG_DIR / "_torch_calls.so"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr", "-Xcompiler", "-fvisibility=hidden",
]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libvjattn")
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _headers_mtime() -> float:
    hs = list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def _compile(src: Path, obj: Path, ptxas_v: bool) -> str:
    cmd = [_nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, f"-I{INCLUDE}", "-c", str(src), "-o", str(obj)]
    if ptxas_v:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return r.stderr


def _calls_stale() -> bool:
    """Whether _torch_calls.so is missing, older than its sources, or another torch's or
    Python's."""
    newest = max(p.stat().st_mtime for p in (CALLS_SRC, INCLUDE / "vjattn.h"))
    return (not CALLS_PATH.exists() or CALLS_PATH.stat().st_mtime < newest
            or not _native.calls_match())


def _build_calls() -> None:
    import torch
    root = Path(torch.__file__).resolve().parent
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        raise RuntimeError("g++ not found; a C++ compiler is required to build _torch_calls")
    cuda = Path(_nvcc()).resolve().parent.parent / "include"
    inc = [root / "include", root / "include/torch/csrc/api/include", cuda,
           sysconfig.get_paths()["include"]]
    tmp = CALLS_PATH.with_suffix(".so.tmp")
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           f'-DVJ_CALLS_TARGET="{_native.calls_target()}"',
           *(f"-I{i}" for i in inc), str(CALLS_SRC), "-o", str(tmp), f"-L{root / 'lib'}",
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {CALLS_SRC.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, CALLS_PATH)


def build(force: bool = False, ptxas_v: bool = False, verbose: bool = False) -> Path:
    BUILD_DIR.mkdir(exist_ok=True)
    hdr_t = _headers_mtime()
    jobs = []
    objs = []
    for src in sources():
        obj = BUILD_DIR / (src.stem + ".o")
        objs.append(obj)
        stale = (force or ptxas_v or not obj.exists()
                 or obj.stat().st_mtime < max(src.stat().st_mtime, hdr_t))
        if stale:
            jobs.append((src, obj))
    stale_calls = force or _calls_stale()
    with cf.ThreadPoolExecutor(max_workers=8) as ex:
        calls = ex.submit(_build_calls) if stale_calls else None
        if jobs:
            futs = {ex.submit(_compile, s, o, ptxas_v): s for s, o in jobs}
            for f in cf.as_completed(futs):
                log = f.result()
                if (verbose or ptxas_v) and log:
                    print(f"--- {futs[f].name}\n{log}", file=sys.stderr)
        if calls is not None:
            calls.result()
    newest = max(o.stat().st_mtime for o in objs)
    if force or jobs or not LIB_PATH.exists() or LIB_PATH.stat().st_mtime < newest:
        tmp = LIB_PATH.with_suffix(".so.tmp")
        cmd = [_nvcc(), *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objs)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB_PATH)
    return LIB_PATH


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-v", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, ptxas_v=a.ptxas_v, verbose=a.verbose))


if __name__ == "__main__":
    main()
