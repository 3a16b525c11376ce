"""Builds libdressi_b200.so in-tree with nvcc for sm_100a, and the torch
binding of its learning operators (_torch_binding.so) with g++.

    python -m opendressi_b200.build        # or opendressi_b200.build.build()

-fmad=false is required, not a tuning choice: the rasterizer's triangle-ID,
coverage and distance outputs are bit-exact with the reference CPU code only
when every multiply and add is rounded separately, as on x86-64 SSE. The
default -prec-div / -prec-sqrt / -ftz=false keep IEEE division, square root
and denormals.
"""

from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libdressi_b200.so")
BINDING_SOURCE = os.path.join(CSRC, "torch_binding.cpp")
BINDING = os.path.join(HERE, "_torch_binding.so")
SOURCES = ["capi.cu", "soft_raster.cu", "silhouette.cu", "hard_raster.cu",
           "fit.cu", "noalloc.cu",
           "antialias.cu", "texture.cu", "interp.cu", "regularize.cu",
           "ibl.cu", "pbr.cu", "faces.cu", "paper.cu", "paper_pixel.cu",
           "group_norm.cu", "adamw.cu",
           "graph_ops.cpp", "graph_exec.cu", "graph_ad.cu"]
HEADERS = ["common.h", "exact.cuh", "kernels.h", "raster_soft.cuh",
           "graph.h", "graph_exec.h"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-fmad=false", "-prec-div=true", "-prec-sqrt=true", "-ftz=false",
    "-Xcompiler", "-fPIC,-O2",
    "--expt-relaxed-constexpr",
]


# The C5 shading (pbr.cu), the paper path's per-pixel chain (paper_pixel.cu)
# and the group normalisation (group_norm.cu) have a tolerance contract, not a
# bit-exact one: they contract a * b + c into FMAs and use the fast (<= 2 ulp)
# division, as GPU shader compilers do. Every other translation unit keeps the
# strict flags above (the raster and IBL ops are bit-exact with the reference).
FILE_FLAGS = {"pbr.cu": {"-fmad=false": "-fmad=true",
                         "-prec-div=true": "-prec-div=false"},
              "paper_pixel.cu": {"-fmad=false": "-fmad=true",
                                 "-prec-div=true": "-prec-div=false"},
              "group_norm.cu": {"-fmad=false": "-fmad=true",
                                "-prec-div=true": "-prec-div=false"}}


def flags_for(src: str) -> list[str]:
    sub = FILE_FLAGS.get(src, {})
    # DRESSI_NVCC_DEFINES: extra -D tuning macros of the kernels (for
    # instance "-DDRESSI_WARP_SORT=64"); empty in a normal build
    extra = os.environ.get("DRESSI_NVCC_DEFINES", "").split()
    return [sub.get(f, f) for f in NVCC_FLAGS] + extra


def nvcc() -> str:
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin",
                        "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def _older(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    deps = deps + [os.path.join(ROOT, "include", "dressi_b200.h"),
                   os.path.abspath(__file__)]
    return any(os.path.getmtime(p) > t for p in deps if os.path.exists(p))


def _stale() -> bool:
    return _older(LIB, [os.path.join(CSRC, f) for f in SOURCES + HEADERS])


def _binding_command() -> list[str]:
    """g++ for the torch binding: an extension module over torch's headers
    and libdressi_b200.so (found beside it)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    lib = cpp_extension.library_paths()
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
            "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_torch_binding",
            "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI,
            *[f"-isystem{p}" for p in cpp_extension.include_paths()],
            f"-isystem{os.path.join(cuda, 'include')}",
            f"-isystem{sysconfig.get_paths()['include']}", BINDING_SOURCE,
            "-o", BINDING, *[f"-L{p}" for p in lib], f"-L{HERE}",
            "-l:libdressi_b200.so", "-Wl,-rpath,$ORIGIN", "-lc10",
            "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch",
            "-ltorch_python"]


def _build_binding(force: bool, verbose: bool) -> None:
    if not force and not _older(BINDING, [BINDING_SOURCE]):
        return
    cmd = _binding_command()
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    out = subprocess.run(cmd, capture_output=True, text=True)
    if out.returncode != 0:
        raise RuntimeError("g++ failed on torch_binding.cpp:\n" + out.stdout +
                           out.stderr)


def build(force: bool = False, verbose: bool = False, jobs: int = 8) -> str:
    """Compiles every translation unit, links the shared library and the
    torch binding over it."""
    _build_library(force, verbose, jobs)
    _build_binding(force, verbose)
    return LIB


def _build_library(force: bool, verbose: bool, jobs: int) -> None:
    if not force and not _stale():
        return
    obj_dir = os.path.join(HERE, "_build")
    os.makedirs(obj_dir, exist_ok=True)
    objs, procs = [], []
    for src in SOURCES:
        obj = os.path.join(obj_dir, os.path.splitext(src)[0] + ".o")
        objs.append(obj)
        cmd = [nvcc(), *flags_for(src), "-c", os.path.join(CSRC, src), "-o",
               obj]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE,
                                            stderr=subprocess.STDOUT)))
        if len(procs) >= jobs:
            _wait(procs.pop(0))
    for p in procs:
        _wait(p)
    link = [nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared",
            "-o", LIB, *objs, "-lcudart"]
    out = subprocess.run(link, capture_output=True, text=True)
    if out.returncode != 0:
        raise RuntimeError("link failed:\n" + out.stdout + out.stderr)


def _wait(item):
    src, p = item
    out, _ = p.communicate()
    if p.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{out.decode()}")


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
