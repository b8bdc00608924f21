"""Builds libg4b_attn.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a.

Usage: ``python -m g4b_b200.build [--force] [--verbose]``.  nvcc cross-compiles without a
GPU.  The library lands in ``g4b_b200/lib/libg4b_attn.so``; objects in ``g4b_b200/lib/obj``.
"""
from __future__ import annotations

import concurrent.futures
import hashlib
import importlib.metadata
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIBDIR = PKG / "lib"
LIB = LIBDIR / "libg4b_attn.so"
VIEWS = LIBDIR / "_views.so"           # argument packing for torch tensors (a CPython module)
INCLUDE = PKG.parent / "include"

SOURCES = ["api.cu", "kv_append.cu", "rope_append.cu", "combine.cu", "combine_exchange.cu", "decode.cu", "decode_stream.cu", "decode_static.cu", "tensor_map.cu", "prefill_sm100.cu",
           "page_copy.cu", "rope_packed.cu", "prefill_packed_sm100.cu"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
    "-I", str(INCLUDE),
]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; libg4b_attn.so cannot be built")
    return cand


def _torch_version() -> str:
    """Of the torch that views.cpp is built against; "" where there is none (the library needs none)."""
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return ""


def _digest() -> str:
    h = hashlib.sha256()
    for f in sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.cpp")) + list(INCLUDE.glob("*.h"))):
        h.update(f.name.encode())
        h.update(f.read_bytes())
    h.update(" ".join(NVCC_FLAGS).encode())
    h.update(f"{_torch_version()} {sys.version}".encode())
    return h.hexdigest()


def _build_views() -> bool:
    """The CPython module that packs torch tensors (csrc/views.cpp), against the torch that is installed; False where
    that cannot be built (no g++, no Python headers, a torch without CUDA).  The library needs none of it: without the
    module the Python code of _cabi.py packs."""
    if not _torch_version():
        VIEWS.unlink(missing_ok=True)
        return False
    try:
        _compile_views()
    except Exception as e:      # whatever keeps it from being built, the library does not depend on it
        VIEWS.unlink(missing_ok=True)      # (not one of another torch)
        sys.stderr.write(f"g4b_b200: argument packing stays in Python, {VIEWS.name} was not built: {e}\n")
        return False
    return True


def _compile_views() -> None:
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths

    nvcc_root = Path(_nvcc()).resolve().parents[1]
    libs = Path(torch.__file__).parent / "lib"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-w", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DG4B_BUILT_FOR="{torch.__version__} {sys.version.split()[0]} {sys.implementation.cache_tag}"',
           *[f"-I{d}" for d in include_paths()], f"-I{sysconfig.get_paths()['include']}", f"-I{nvcc_root / 'include'}",
           str(CSRC / "views.cpp"), "-o", str(VIEWS), f"-L{libs}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for views.cpp:\n{res.stdout}\n{res.stderr}")


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every .cu for sm_100a and link the shared library. Returns its path."""
    LIBDIR.mkdir(exist_ok=True)
    objdir = LIBDIR / "obj"
    objdir.mkdir(exist_ok=True)
    stamp = LIBDIR / "build.stamp"
    digest = _digest()
    # (a module that could not be built is not tried again until something changes)
    if not force and LIB.exists() and stamp.exists() and stamp.read_text() == digest + (" views" if VIEWS.exists() else ""):
        return LIB
    nvcc = _nvcc()
    extra = ["-Xptxas", "-v"] if verbose else []

    def compile_one(src: str) -> Path:
        obj = objdir / (Path(src).stem + ".o")
        cmd = [nvcc, *NVCC_FLAGS, *extra, "-c", str(CSRC / src), "-o", str(obj)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{res.stdout}\n{res.stderr}")
        if verbose:
            sys.stderr.write(res.stderr)
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(SOURCES) + 1)) as ex:
        views = ex.submit(_build_views)
        objs = list(ex.map(compile_one, SOURCES))
        views_built = views.result()
    cmd = [nvcc, "-shared", "-o", str(LIB), *map(str, objs), "-cudart", "static"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    stamp.write_text(digest + (" views" if views_built else ""))
    return LIB


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(path)
