"""Build recipe for the in-tree CUDA library ``libmkx.so`` (sm_100a only) and its torch binding ``_mkx_torch.<key>.so``.

    python -m reki_megakernel_b200.build             # libmkx.so
    python -m reki_megakernel_b200.build --traced    # libmkx_trace.so (profiling variant)

nvcc cross-compiles without a GPU; the library lands next to this file so it travels with the
source tree and is the one ``reki_megakernel_b200._lib`` loads.
"""
from __future__ import annotations

import hashlib
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
LIB = PKG / "libmkx.so"
# Profiling variant: the same sources with -DMKX_SUBSTAGE_TRACE (thread 0 of CTAs 0 and 100 stamps
# %globaltimer at numbered points inside each stage); loaded only after _lib.use_traced_build().
TRACE_LIB = PKG / "libmkx_trace.so"
SOURCES = [PKG / "csrc" / "mk_expert.cu", PKG / "csrc" / "mk_prepare.cu", PKG / "csrc" / "mk_mods.cu",
           PKG / "csrc" / "mk_batch.cu", PKG / "csrc" / "mk_copies.cu", PKG / "csrc" / "mk_cache.cu",
           PKG / "csrc" / "mk_attend.cu"]
HEADERS = [PKG / "csrc" / "mkx_device.cuh", PKG / "csrc" / "mkx_tma.cuh", PKG / "csrc" / "mkx_half.cuh",
           PKG / "csrc" / "mkx_attend.cuh", PKG / "csrc" / "mkx_join.h", PKG / "csrc" / "mkx_pdl.cuh", PKG / "csrc" / "mkx_cache_host.h", ROOT / "include" / "mkx.h",
           ROOT / "include" / "mkx_prepare.h", ROOT / "include" / "mkx_mods.h", ROOT / "include" / "mkx_batch.h",
           ROOT / "include" / "mkx_cache.h"]
# The episode cache's entry points for torch tensors (host code; reaches libmkx.so by address).
TORCH_SOURCES = [PKG / "csrc" / "mk_torch.cpp", ROOT / "include" / "mkx.h", ROOT / "include" / "mkx_cache.h"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libmkx.so")
    return cand


def stale(lib: Path | None = None) -> bool:
    lib = lib or LIB
    if not lib.exists():
        return True
    t = lib.stat().st_mtime
    return any(p.stat().st_mtime > t for p in SOURCES + HEADERS)


def _digest(*parts) -> str:
    h = hashlib.sha256()
    for p in parts:
        h.update(p.read_bytes() if isinstance(p, Path) else str(p).encode())
        h.update(b"\0")
    return h.hexdigest()


def cache_key() -> int:
    """The episode cache's structs as a number: what include/mkx_cache.h says. Both libraries carry it, since one hands the
    other raw structs."""
    return int(_digest(ROOT / "include" / "mkx_cache.h")[:15], 16)


def torch_lib() -> Path:
    """The torch binding of these sources, this torch and this Python: another one has another name, so that none is loaded
    in place of one that cannot be built."""
    key = _digest(*TORCH_SOURCES, importlib.metadata.version("torch"), sysconfig.get_config_var("SOABI"))
    return PKG / f"_mkx_torch.{key[:12]}.so"


def build(force: bool = False, verbose: bool = False, traced: bool = False) -> Path:
    lib = TRACE_LIB if traced else LIB
    if not force and not stale(lib):
        return lib
    tmp = lib.with_suffix(f".so.tmp{os.getpid()}")
    cmd = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-shared",
           *(["-DMKX_SUBSTAGE_TRACE"] if traced else []), f"-DMKX_CACHE_KEY={cache_key():#x}ull",
           "-I", str(ROOT / "include"), "-I", str(PKG / "csrc"), "-o", str(tmp), *map(str, SOURCES)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    if verbose:
        print(r.stderr, file=sys.stderr)
    os.replace(tmp, lib)
    return lib


def build_torch(force: bool = False) -> Path:
    """Compiles the torch binding with the host compiler against the headers of the installed torch."""
    lib = torch_lib()
    if not force and lib.exists():
        return lib
    gxx = shutil.which("g++")
    spec = importlib.util.find_spec("torch")
    if gxx is None or spec is None:
        raise RuntimeError(f"g++ and torch are required to build {lib.name}")
    torch = Path(spec.submodule_search_locations[0])
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = lib.with_suffix(f".so.tmp{os.getpid()}")
    cmd = [gxx, "-O2", "-std=c++17", "-fPIC", "-shared", f"-DMKX_CACHE_KEY={cache_key():#x}ull", "-I", str(torch / "include"), "-I", sysconfig.get_paths()["include"],
           "-I", str(cuda / "include"), "-I", str(ROOT / "include"), "-o", str(tmp), str(TORCH_SOURCES[0]),
           "-L", str(torch / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, lib)
    for old in PKG.glob("_mkx_torch*.so"):  # of other sources
        if old != lib:
            old.unlink(missing_ok=True)
    return lib


if __name__ == "__main__":
    print(build_torch(force="--force" in sys.argv))
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv, traced="--traced" in sys.argv))
