"""Build librotatek_b200.so (the C-ABI library) for sm_100a with nvcc.

    python -m rotatek_b200.csrc.build [--verbose]

The library lands next to the package (rotatek_b200/librotatek_b200.so) so a
snapshot of the source tree carries it.  The CUDA runtime is linked
statically: the library does not depend on which libcudart the host process
(e.g. torch) has loaded.  cuTensorMapEncodeTiled is resolved at run time
through cudaGetDriverEntryPointByVersion, so there is no -lcuda.  Beside it lands
rotatek_b200/_calls.so, the CPython module that calls the shared-prefix entry
points without ctypes.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

CSRC = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(CSRC)
REPO = os.path.dirname(PKG)
LIB_NAME = "librotatek_b200.so"
CALLS_NAME = "_calls.so"          # CPython module over the C ABI (calls.c)
SOURCES = ["capi.cu", "decode_tc.cu", "decode_simt.cu", "decode_static.cu", "quant_fp8.cu", "spark_pack.cu", "cov_tc.cu", "kproj_tc.cu", "eigen.cu",
           "rotate.cu", "selftest.cu", "capi_shared.cu", "shared_simt.cu", "shared_prefix.cu", "shared_text.cu", "shared_merge.cu", "text_cache.cu", "verify.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC)")


def build(verbose: bool = False, out_dir: str = PKG) -> str:
    out = os.path.join(out_dir, LIB_NAME)
    obj_dir = os.path.join(REPO, "_build")
    os.makedirs(obj_dir, exist_ok=True)
    flags = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
                    "--expt-relaxed-constexpr", "-I", os.path.join(REPO, "include")]
    if verbose:
        flags += ["-Xptxas", "-v"]
    objs = []
    for src in SOURCES:
        obj = os.path.join(obj_dir, src.replace(".cu", ".o"))
        cmd = [nvcc()] + flags + ["-c", os.path.join(CSRC, src), "-o", obj]
        subprocess.run(cmd, check=True)
        objs.append(obj)
    tmp = out + ".tmp"
    subprocess.run([nvcc()] + ARCH + ["-shared", "-cudart", "static", "-o", tmp] + objs, check=True)
    os.replace(tmp, out)
    build_calls(out_dir)
    return out


def build_calls(out_dir: str = PKG) -> str:
    """The Python module of direct calls: a C file against Python.h and torch's copy of dlpack.h."""
    out = os.path.join(out_dir, CALLS_NAME)
    cc = os.environ.get("CC") or shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        raise RuntimeError("no C compiler found (set CC)")
    subprocess.run([cc, "-O2", "-std=c11", "-Wall", "-shared", "-fPIC", "-I", sysconfig.get_paths()["include"],
                    "-I", os.path.join(importlib.util.find_spec("torch").submodule_search_locations[0], "include"),
                    os.path.join(CSRC, "calls.c"), "-o", out + ".tmp", "-ldl"], check=True)
    os.replace(out + ".tmp", out)
    return out


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true", help="print ptxas register / smem usage")
    args = ap.parse_args()
    print(build(verbose=args.verbose))


if __name__ == "__main__":
    sys.exit(main())
