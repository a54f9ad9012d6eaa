"""Builds libshellcache.so (the C ABI) in-tree with nvcc for sm_100a only, and beside it
_fastpath.so, the callers of the group-decode operators (needs torch and Python headers)."""

from __future__ import annotations

import os
import shutil
import subprocess
import sysconfig
import warnings
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
CSRC = PACKAGE / "csrc"
LIBRARY = PACKAGE / "libshellcache.so"
FASTPATH = PACKAGE / "_fastpath.so"
SOURCES = ("status.cu", "gdn_decode.cu", "gdn_front.cu", "gdn_chunk.cu", "paged_kv.cu",
           "paged_attention.cu", "paged_q8.cu", "exchange.cu", "shared_prefix.cu", "rotary.cu",
           "beam.cu")
ARCH = ("-gencode", "arch=compute_100a,code=sm_100a")


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(found):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build shellcache")
    return found


def _stale() -> bool:
    if not LIBRARY.exists():
        return True
    built = LIBRARY.stat().st_mtime
    inputs = [CSRC / name for name in SOURCES] + list(CSRC.glob("*.cuh"))
    inputs.append(PACKAGE.parent / "include" / "shellcache.h")
    return any(p.stat().st_mtime > built for p in inputs if p.exists())


def _build_fastpath(force: bool, verbose: bool) -> None:
    """Compile the callers (csrc/fastpath.cpp) against torch; they link the library. They are
    optional: where g++, torch, its CUDA headers or Python's are missing, a warning says so, callers of
    an older build are removed, and the Python wrappers make the calls."""
    inputs = [CSRC / "fastpath.cpp", PACKAGE.parent / "include" / "shellcache.h", Path(__file__)]
    if not force and FASTPATH.exists() and all(p.stat().st_mtime <= FASTPATH.stat().st_mtime
                                               for p in inputs):
        return
    tmp = FASTPATH.with_suffix(".so.tmp")
    try:
        import torch

        base = Path(torch.__file__).resolve().parent
        cuda = Path(nvcc()).resolve().parent.parent
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
               f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
               f'-DSC_TORCH_VERSION="{torch.__version__}"',
               f"-I{base}/include", f"-I{base}/include/torch/csrc/api/include",
               f"-I{sysconfig.get_paths()['include']}", f"-I{cuda}/include", str(inputs[0]),
               "-o", str(tmp), f"-L{PACKAGE}", "-l:libshellcache.so", f"-L{base}/lib", "-lc10",
               "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
        if verbose:
            print(" ".join(cmd))
        proc = subprocess.run(cmd, capture_output=True, text=True)
        failed = f"g++ failed ({proc.returncode}):\n{proc.stderr[-4000:]}" if proc.returncode else None
    except (ImportError, OSError, RuntimeError) as err:  # RuntimeError: no CUDA toolkit
        failed = f"{type(err).__name__}: {err}"
    if failed is not None:
        FASTPATH.unlink(missing_ok=True)
        warnings.warn(f"the group-decode operators' compiled callers are not built, their Python "
                      f"wrappers will be used: {failed}", stacklevel=2)
        return
    os.replace(tmp, FASTPATH)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every kernel source into one shared library next to this file."""
    if not force and not _stale():
        _build_fastpath(False, verbose)
        return LIBRARY
    tmp = LIBRARY.with_suffix(".so.tmp")
    cmd = [
        nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
        "-Xcompiler", "-fPIC,-O3", "-shared", "-o", str(tmp),
        *[str(CSRC / name) for name in SOURCES],
    ]
    if verbose:
        print(" ".join(cmd))
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{proc.stderr[-4000:]}")
    os.replace(tmp, LIBRARY)
    _build_fastpath(force, verbose)
    return LIBRARY


if __name__ == "__main__":
    print(build(force=True, verbose=True))
