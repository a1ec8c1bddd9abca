"""Builds the native libraries in-tree.

* ``libmlb200.so``   — the sm_100a kernels, the decode runtime and the C ABI of
  include/mlb200.h (nvcc, ``-gencode arch=compute_100a,code=sm_100a``), linked
  against NCCL for tensor parallelism.
* ``libmlb_synth.so`` — the CPU side of the seeded synthetic-weight generator
  (g++, no CUDA).
* ``_calls-*.so``    — the int8 layer's calls on torch tensors (g++, torch's headers),
  over libmlb200.so; named after its sources and the torch and Python it is for.

All land next to this file so they travel with the source tree.
"""
from __future__ import annotations

import glob
import hashlib
import importlib.util
import os
import re
import subprocess
import sys
import sysconfig
import threading

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libmlb200.so")
SYNTH_LIB = os.path.join(HERE, "libmlb_synth.so")

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nccl_dirs():
    """NCCL headers and library: the pip package torch uses, else the system one."""
    purelib = sysconfig.get_paths()["purelib"]
    pkg = os.path.join(purelib, "nvidia", "nccl")
    inc, lib = os.path.join(pkg, "include"), os.path.join(pkg, "lib")
    if os.path.exists(os.path.join(inc, "nccl.h")) and os.path.exists(os.path.join(lib, "libnccl.so.2")):
        return inc, lib
    return "/usr/include", "/usr/lib/x86_64-linux-gnu"


def _stale(target: str, sources) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def build_cuda(force: bool = False, verbose: bool = False) -> str:
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    deps = srcs + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + [
        os.path.join(ROOT, "include", "mlb200.h")]
    if not force and not _stale(LIB, deps):
        return LIB
    inc, lib = _nccl_dirs()
    # one nvcc per translation unit, in parallel, then one link
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    flags = [*ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
             "--expt-relaxed-constexpr", "-I", inc, "-I", os.path.join(ROOT, "include")]
    if verbose:
        flags.insert(0, "-Xptxas=-v")
    objs = [os.path.join(objdir, os.path.basename(s) + ".o") for s in srcs]

    def compile_one(pair):
        src, obj = pair
        subprocess.run([NVCC, *flags, "-c", "-o", obj, src], check=True)

    from concurrent.futures import ThreadPoolExecutor

    with ThreadPoolExecutor(max_workers=min(len(srcs), os.cpu_count() or 4)) as ex:
        list(ex.map(compile_one, zip(srcs, objs)))
    subprocess.run([NVCC, *ARCH, "-shared", "-o", LIB + ".tmp", *objs, "-L", lib,
                    "-l:libnccl.so.2", "-Xlinker", "-rpath=" + lib], check=True)
    os.replace(LIB + ".tmp", LIB)
    return LIB


def build_synth(force: bool = False) -> str:
    src = os.path.join(CSRC, "synth_host.cc")
    deps = [src, os.path.join(CSRC, "synth.h")]
    if not force and not _stale(SYNTH_LIB, deps):
        return SYNTH_LIB
    cmd = ["g++", "-O3", "-std=c++17", "-fPIC", "-shared", "-ffp-contract=off", "-pthread",
           "-o", SYNTH_LIB + ".tmp", src]
    subprocess.run(cmd, check=True)
    os.replace(SYNTH_LIB + ".tmp", SYNTH_LIB)
    return SYNTH_LIB


def _torch_dir():
    """Where torch with CUDA is installed, or None."""
    spec = importlib.util.find_spec("torch")
    at = os.path.dirname(spec.origin) if spec and spec.origin else ""
    return at if os.path.exists(os.path.join(at, "lib", "libc10_cuda.so")) else None


def _torch_version(torch: str) -> str:
    """Of the torch in a directory, without importing it."""
    with open(os.path.join(torch, "version.py")) as f:
        found = re.search(r"__version__ = ['\"]([^'\"]+)", f.read())
    return found.group(1) if found else "unknown"


def calls_path() -> str:
    """Where the calls on torch tensors belong: built from other sources, or for another
    torch or Python, they have another name."""
    torch = _torch_dir()
    if torch is None:
        raise RuntimeError("calls on torch tensors need torch with CUDA")
    h = hashlib.sha1()
    for path in (os.path.join(CSRC, "torch_calls.cc"), os.path.join(ROOT, "include", "mlb200.h")):
        with open(path, "rb") as f:
            h.update(f.read())
    h.update(f"{_torch_version(torch)} {sysconfig.get_config_var('SOABI')}".encode())
    return os.path.join(HERE, f"_calls-{h.hexdigest()[:12]}.so")


def _calls_headers(torch: str) -> bool:
    return all(os.path.exists(os.path.join(*at)) for at in (
        (torch, "include", "ATen", "ATen.h"), (sysconfig.get_paths()["include"], "Python.h")))


def build_calls(force: bool = False) -> str:
    path = calls_path()
    if not force and os.path.exists(path):
        return path
    torch = _torch_dir()
    lib = os.path.join(torch, "lib")
    # processes and threads that build at once stay apart
    made = f"{path}.{os.getpid()}.{threading.get_ident()}.tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-o", made,
           os.path.join(CSRC, "torch_calls.cc"),
           "-I", os.path.join(torch, "include"),
           "-I", os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           "-I", os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include"),
           "-I", sysconfig.get_paths()["include"],
           "-L", lib, "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
           "-L", HERE, "-l:libmlb200.so", "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + lib]
    try:
        subprocess.run(cmd, check=True)
        os.replace(made, path)
    finally:
        if os.path.exists(made):
            os.remove(made)
    return path


def build(force: bool = False, verbose: bool = False) -> None:
    build_synth(force)
    build_cuda(force, verbose)
    torch = _torch_dir()
    if torch and _calls_headers(torch):  # without them the Python forms do the calls' work
        build_calls(force)


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
