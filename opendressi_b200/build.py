"""Builds libdressi_b200.so in-tree with nvcc for sm_100a, and the torch
binding of its learning operators (_torch_binding.so) with g++.

    python -m opendressi_b200.build        # or opendressi_b200.build.build()
    python -m opendressi_b200.build --library    # without the torch binding

-fmad=false is required, not a tuning choice: the rasterizer's triangle-ID,
coverage and distance outputs are bit-exact with the reference CPU code only
when every multiply and add is rounded separately, as on x86-64 SSE. The
default -prec-div / -prec-sqrt / -ftz=false keep IEEE division, square root
and denormals.
"""

from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libdressi_b200.so")
BINDING_SOURCE = os.path.join(CSRC, "torch_binding.cpp")
BINDING = os.path.join(HERE, "_torch_binding.so")
OBJ_DIR = os.path.join(HERE, "_build")
BINDING_STAMP = os.path.join(OBJ_DIR, "torch_binding.txt")
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


def _torch_version() -> str | None:
    """The installed torch's version; None where there is none."""
    if importlib.util.find_spec("torch") is None:
        return None
    return importlib.metadata.version("torch")


def _binding_commands() -> tuple[list[str], list[str]]:
    """g++ to compile and to link the torch binding: an extension module over
    torch's headers and libdressi_b200.so (found beside it)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    obj = os.path.join(OBJ_DIR, "torch_binding.o")
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden",
             "-DTORCH_EXTENSION_NAME=_torch_binding",
             "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI,
             *[f"-isystem{p}" for p in cpp_extension.include_paths()],
             f"-isystem{os.path.join(cuda, 'include')}",
             f"-isystem{sysconfig.get_paths()['include']}", "-c",
             BINDING_SOURCE, "-o", obj],
            ["g++", "-shared", "-o", BINDING, obj,
             *[f"-L{p}" for p in cpp_extension.library_paths()], f"-L{HERE}",
             "-l:libdressi_b200.so", "-Wl,-rpath,$ORIGIN", "-lc10",
             "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch",
             "-ltorch_python"])


def _binding_stamp() -> str:
    """What a binding was built for: it loads into no other torch."""
    return f"torch {_torch_version()}, {sys.implementation.cache_tag}\n"


def _binding_stale() -> bool:
    try:
        with open(BINDING_STAMP) as f:
            if f.read() != _binding_stamp():
                return True
    except OSError:
        return True
    return _older(BINDING, [BINDING_SOURCE])


def build(force: bool = False, verbose: bool = False, jobs: int = 8,
          binding: bool = True) -> str:
    """Compiles every translation unit and links the shared library and, where
    torch is installed and `binding` is not False, the torch binding over it
    (the library itself needs neither torch nor its headers)."""
    link = compiled = None
    if binding and _torch_version() is None:
        print("torch is not installed: its binding of the learning operators "
              "is left out", file=sys.stderr)
    elif binding and (force or _binding_stale()):
        compile_, link = _binding_commands()
        os.makedirs(OBJ_DIR, exist_ok=True)
        if verbose:
            print(" ".join(compile_), file=sys.stderr)
        compiled = subprocess.Popen(compile_, stdout=subprocess.PIPE,
                                    stderr=subprocess.STDOUT)
    try:
        _build_library(force, verbose, jobs)
    except BaseException:
        if compiled:
            compiled.kill()
            compiled.communicate()
        raise
    if link:
        _wait(("torch_binding.cpp", compiled))
        out = subprocess.run(link, capture_output=True, text=True)
        if out.returncode != 0:
            raise RuntimeError("linking the torch binding failed:\n" +
                               out.stdout + out.stderr)
        with open(BINDING_STAMP, "w") as f:
            f.write(_binding_stamp())
    return LIB


def _build_library(force: bool, verbose: bool, jobs: int) -> None:
    if not force and not _stale():
        return
    os.makedirs(OBJ_DIR, exist_ok=True)
    objs, procs = [], []
    for src in SOURCES:
        obj = os.path.join(OBJ_DIR, os.path.splitext(src)[0] + ".o")
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
        raise RuntimeError(f"compiling {src} failed:\n{out.decode()}")


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True,
                binding="--library" not in sys.argv))
