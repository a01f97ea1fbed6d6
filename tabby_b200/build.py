"""Build the shared libraries in-tree with nvcc for sm_100a.

    python -m tabby_b200.build        # -> tabby_b200/lib/

libtabbysample.so (include/tabby_sample.h) is the sampler, libtabbydecode.so
(include/tabby_decode.h) the decode operators for several hypotheses a sequence. Both are
plain C-ABI shared objects that do not link against torch. CUDA's runtime is linked
statically so they only need the driver. tabby_decode_torch.so is the Python side of the
second on torch tensors (decode.py), an extension module built with g++ against torch; where
either is missing it is left out with a note, since the libraries need neither.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIBDIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIBDIR, "libtabbysample.so")
SOURCES = ["sampler_kernels.cu", "capi.cu", "noalloc.cu", "softmax_rows.cu", "lmhead.cu",
           "exchange.cu"]
DECODE_LIB = os.path.join(LIBDIR, "libtabbydecode.so")
DECODE_SOURCES = ["decode_capi.cu", "beam.cu", "states.cu", "tree_attention.cu"]
DECODE_TORCH = os.path.join(LIBDIR, "tabby_decode_torch.so")
HEADERS = ["decode_internal.h", "finalize.cuh", "js_math.cuh", "sampler_internal.h", "sm100.cuh",
           "warp_sort.cuh"]

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-ffp-contract=off,-fvisibility=hidden",
    "-Xptxas", "-v",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale(lib: str, sources: list) -> bool:
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    deps = [os.path.join(CSRC, f) for f in sources + HEADERS]
    deps += [os.path.join(ROOT, "include", h) for h in ("tabby_sample.h", "tabby_decode.h")]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _run(cmd: list, what: str) -> str:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what}:\n{r.stdout}\n{r.stderr}")
    return r.stderr


def _build_lib(lib_path: str, sources: list, verbose: bool, defines: tuple) -> None:
    libdir = os.path.dirname(lib_path)
    os.makedirs(libdir, exist_ok=True)
    objs = [os.path.join(libdir, os.path.splitext(src)[0] + ".o") for src in sources]
    cmds = [[nvcc(), *ARCH, *NVCC_FLAGS, *[f"-D{d}" for d in defines],
             "-I", os.path.join(ROOT, "include"), "-I", CSRC,
             "-c", os.path.join(CSRC, src), "-o", obj] for src, obj in zip(sources, objs)]
    with ThreadPoolExecutor(max_workers=len(cmds)) as pool:  # a process a source
        for err in pool.map(_run, cmds, [f"nvcc failed for {src}" for src in sources]):
            if verbose:
                sys.stderr.write(err)
    tmp = lib_path + ".tmp"
    _run([nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", tmp, *objs,
          "-Xlinker", "--exclude-libs,ALL"], "link failed")
    os.replace(tmp, lib_path)
    for o in objs:
        os.remove(o)


def _build_torch() -> None:
    import sysconfig

    gxx = shutil.which("g++")
    missing = "" if gxx else "g++"
    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError:
        missing = "torch"
    else:
        if torch.version.cuda is None:
            missing = "torch with CUDA"
    if missing:
        sys.stderr.write(f"{missing} is missing: {os.path.basename(DECODE_TORCH)} is not built "
                         "(tabby_b200.decode needs it)\n")
        return
    libs = cpp_extension.library_paths()
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    includes = [os.path.join(ROOT, "include"), os.path.join(cuda, "include"),
                sysconfig.get_paths()["include"], *cpp_extension.include_paths()]
    tmp = DECODE_TORCH + ".tmp"
    _run([gxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
          "-DTORCH_EXTENSION_NAME=tabby_decode_torch",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          *[f"-I{i}" for i in includes], os.path.join(CSRC, "decode_torch.cpp"), "-o", tmp,
          f"-L{LIBDIR}", "-l:libtabbydecode.so", *[f"-L{p}" for p in libs], "-ltorch",
          "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN"],
         "g++ failed for decode_torch.cpp")
    os.replace(tmp, DECODE_TORCH)


def build(force: bool = False, verbose: bool = False, out: str | None = None,
          defines: tuple = ()) -> str:
    """Compile the libraries in-tree and return the sampler's path; with `out`, only
    SOURCES into that path. `defines` adds -D flags (e.g. TABBY_CHECKS=1 for the
    self-checking debug build)."""
    if out is not None:
        _build_lib(out, SOURCES, verbose, defines)
        return out
    for lib_path, sources in ((LIB, SOURCES), (DECODE_LIB, DECODE_SOURCES)):
        if force or _stale(lib_path, sources):
            _build_lib(lib_path, sources, verbose, defines)
    if force or _stale(DECODE_TORCH, ["decode_torch.cpp"]):
        _build_torch()
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
