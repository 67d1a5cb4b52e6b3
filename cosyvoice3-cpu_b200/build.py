"""Compile ``csrc/*.cu`` into the in-tree ``libcv3cuda.so`` for sm_100a.

``csrc/bind/*.cpp`` become Python extension modules next to it, for hosts with PyTorch (the short
way of its callers to some entries; the library itself needs no GPU framework, and one that does not
compile is a warning).

Each translation unit is compiled by nvcc (in parallel, skipped when its object
is newer than its sources and headers) and linked with ``nvcc -shared``.  The
library lands next to this file so it travels with the source tree; the
Python host (:mod:`._lib`) loads it from there.

    python cosyvoice3-cpu_b200/build.py [--force] [-j N]
"""

from __future__ import annotations

import argparse
import glob
import os
import subprocess
import sys
import warnings
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
LIB = os.path.join(HERE, "libcv3cuda.so")

NVCC = os.environ.get("NVCC", "nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-I", CSRC, "-I", INCLUDE]


def _deps() -> float:
    """Newest mtime among headers (any header change rebuilds everything)."""
    hs = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def _compile(src: str, force: bool, hdr_time: float, extra) -> str:
    obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), hdr_time):
        return obj
    cmd = [NVCC, *ARCH, *FLAGS, *extra, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {os.path.basename(src)}:\n{r.stdout}\n{r.stderr}")
    return obj


def bind_path(src: str) -> str:
    """The extension module of ``csrc/bind/*.cpp`` for the installed PyTorch and the running Python, whose versions are
    in its name: one built against others is not taken for it."""
    from importlib import metadata
    try:
        version = metadata.version("torch")
    except metadata.PackageNotFoundError:
        version = "none"
    return os.path.join(HERE, "_%s.%s-torch-%s.so" % (os.path.basename(src)[:-4], sys.implementation.cache_tag, version))


def _bind(src: str, force: bool) -> str:
    """One extension module against the installed PyTorch (skipped where there is none).  Returns what the compiler
    says where it fails: without the module its callers take their long way."""
    import importlib.util
    import sysconfig
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        return ""
    out, torch_dir = bind_path(src), spec.submodule_search_locations[0]
    header = os.path.join(INCLUDE, "cv3cuda.h")
    if not force and os.path.exists(out) and os.path.getmtime(out) >= max(os.path.getmtime(src), os.path.getmtime(header)):
        return ""
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-D_GLIBCXX_USE_CXX11_ABI=1",
           "-I", os.path.join(torch_dir, "include"), "-I", os.path.join(cuda, "include"),
           "-I", sysconfig.get_paths()["include"], src, "-o", out, "-L", os.path.join(torch_dir, "lib"),
           "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda"]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        return f"{os.path.basename(src)} was not built: {e}"
    return "" if r.returncode == 0 else f"{os.path.basename(src)} was not built:\n{r.stdout}\n{r.stderr}"


def build(force: bool = False, jobs: int = 0, extra=()) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    if not srcs:
        raise RuntimeError(f"no CUDA sources under {CSRC}")
    hdr = _deps()
    jobs = jobs or min(len(srcs), os.cpu_count() or 4)
    with ThreadPoolExecutor(jobs) as ex:
        binds = [ex.submit(_bind, s, force) for s in sorted(glob.glob(os.path.join(CSRC, "bind", "*.cpp")))]
        objs = list(ex.map(lambda s: _compile(s, force, hdr, list(extra)), srcs))
        said = [b.result() for b in binds]
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        cmd = [NVCC, *ARCH, "-shared", "-o", LIB, *objs, "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    for text in filter(None, said):
        warnings.warn(text)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", type=int, default=0)
    ap.add_argument("--xptxas-v", action="store_true", help="print register/smem usage")
    a = ap.parse_args()
    extra = ["-Xptxas", "-v"] if a.xptxas_v else []
    print(build(force=a.force or a.xptxas_v, jobs=a.j, extra=extra))
    sys.exit(0)
