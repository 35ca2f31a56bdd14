"""Build the sm_100a C-ABI library `libw8a8_b200.so` in-tree with nvcc.

Also the Python binding of the decoding operators, `_decode.so`, with the host compiler
(`csrc/decode_binding.cpp`: torch's C++ API on one side, the C ABI on the other).  Where torch is
not installed there is nothing to bind: only the library is built.

Every `csrc/*.cu` is compiled for `arch=compute_100a,code=sm_100a` (nvcc
cross-compiles without a GPU) into `_build/*.o`, and linked into
`libw8a8_b200.so` next to this file, where `_lib.py` loads it.  Objects are
rebuilt when their source or any header under `csrc/` or `include/` is newer, the binding
also for another torch or Python than it was built for.

usage: python gemma-npu_b200/build.py [--force] [--verbose-ptxas]
"""
import argparse
import glob
import importlib.util
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libw8a8_b200.so")
BINDING = os.path.join(HERE, "_decode.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr",
              f"-I{INCLUDE}"]


def nvcc_path():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put /usr/local/cuda/bin on PATH)")


def _newest(paths):
    return max((os.path.getmtime(p) for p in paths), default=0.0)


def build_binding(force=False, quiet=False):
    """Compile csrc/decode_binding.cpp against this Python and torch; returns its path."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    src = os.path.join(CSRC, "decode_binding.cpp")
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    built_for = f"torch {torch.__version__}, Python {sysconfig.get_config_var('SOABI')}, C++11 ABI {abi}\n"
    note = os.path.join(BUILD, "decode_binding.txt")
    if not force and os.path.exists(BINDING) and os.path.exists(note) and open(note).read() == built_for and (
            os.path.getmtime(BINDING) >= max(os.path.getmtime(src), _newest(glob.glob(os.path.join(INCLUDE, "*.h"))))):
        return BINDING
    os.makedirs(BUILD, exist_ok=True)
    if not quiet:
        print("[build] decode_binding.cpp", flush=True)
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include")
    dirs = [*include_paths(), cuda, sysconfig.get_paths()["include"]]
    tmp = BINDING + ".tmp"
    # The compiler that nvcc links with: a module with a libstdc++ of its own in it must not meet
    # torch's.
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-w",
                    f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
                    *(f"-isystem{d}" for d in dirs), src, "-o", tmp, *(f"-L{d}" for d in library_paths()),
                    "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"], check=True)
    os.replace(tmp, BINDING)
    with open(note, "w") as f:
        f.write(built_for)
    return BINDING


def build(force=False, verbose_ptxas=False, quiet=False):
    """Compile and link; returns the path of the shared library."""
    os.makedirs(BUILD, exist_ok=True)
    nvcc = nvcc_path()
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    hdr_time = _newest(headers)
    objs, stale = [], []
    for src in sources:
        obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if not force and os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), hdr_time):
            continue
        cmd = [nvcc, *ARCH, *NVCC_FLAGS, "-c", src, "-o", obj]
        if verbose_ptxas:
            cmd.insert(1, "-Xptxas=-v")
        stale.append((src, cmd))

    def compile_one(job):
        if not quiet:
            print("[build]", os.path.basename(job[0]), flush=True)
        subprocess.run(job[1], check=True)

    with ThreadPoolExecutor(max(1, os.cpu_count() or 1)) as pool:
        list(pool.map(compile_one, stale))
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < _newest(objs):
        tmp = LIB + ".tmp"
        subprocess.run([nvcc, *ARCH, "-shared", "-o", tmp, *objs], check=True)
        os.replace(tmp, LIB)
        if not quiet:
            print("[build] linked", LIB, flush=True)
    if importlib.util.find_spec("torch") is not None:
        build_binding(force=force, quiet=quiet)
    elif not quiet:
        print("[build] no torch: without the Python binding of the decoding operators", flush=True)
    return LIB


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose-ptxas", action="store_true", help="print registers/spills per kernel")
    a = ap.parse_args(argv)
    build(force=a.force, verbose_ptxas=a.verbose_ptxas)


if __name__ == "__main__":
    sys.exit(main())
