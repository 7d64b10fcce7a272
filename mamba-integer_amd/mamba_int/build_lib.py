"""Builds libmamba_int.so (hipcc, gfx950) in-tree, next to this package, and the module
of the float operators' calls (host C++ against torch) in it.  The library needs hipcc
alone; without torch, a C++ compiler or Python's headers the module is left out."""
from __future__ import annotations

import concurrent.futures
import glob
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile

PKG_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
REPO = os.path.dirname(PKG_ROOT)
CSRC = os.path.join(PKG_ROOT, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB_PATH = os.path.join(PKG_ROOT, "libmamba_int.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CALLS_PATH = os.path.join(PKG_ROOT, "mamba_int", "_float_calls.so")
CXX = os.environ.get("CXX", "g++")
ARCH = "gfx950"

FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    "-Wall", "-Wno-unused-function", "-Wno-unused-variable",
    # packed fp32 VALU forms stay out of every kernel (no v_pk_*_f32)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def sources() -> list:
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def _run(cmd: list, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    errs = "\n".join(l for l in (res.stdout + res.stderr).splitlines()
                     if "packed-fp32-ops" not in l)
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({res.returncode}): {' '.join(cmd)}\n{errs}")
    if verbose and errs.strip():
        print(errs, file=sys.stderr)


def calls_missing() -> list:
    """What the calls' module would need here and does not find."""
    import importlib.util
    missing = [] if importlib.util.find_spec("torch") else ["torch"]
    if shutil.which(CXX) is None:
        missing.append(CXX)
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        missing.append("Python.h")
    return missing


def calls_command(out: str) -> list:
    """g++ of csrc/float_calls.cpp, a Python module that takes torch's tensors."""
    import torch
    root = os.path.dirname(torch.__file__)
    inc, lib = os.path.join(root, "include"), os.path.join(root, "lib")
    return [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}", f"-I{inc}",
            f"-I{os.path.join(inc, 'torch', 'csrc', 'api', 'include')}", f"-I{sysconfig.get_paths()['include']}",
            os.path.join(CSRC, "float_calls.cpp"), "-o", out, f"-L{lib}", f"-Wl,-rpath,{lib}", "-ltorch_python",
            "-ltorch_cpu", "-lc10"]


def build(verbose: bool = False) -> str:
    """Compiles every source to an object in parallel (each file's kernels are
    self-contained: no relocatable device code), then links the library; beside
    them, the calls' module.  An error of the module's leaves the library built."""
    srcs = sources()
    missing = calls_missing()
    with tempfile.TemporaryDirectory(prefix="mamba_int_build_") as tmp:
        objs = [os.path.join(tmp, os.path.basename(s) + ".o") for s in srcs]
        jobs = [[HIPCC, *FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", s, "-o", o] for s, o in zip(srcs, objs)]
        calls = os.path.join(tmp, "calls.so")
        workers = max(1, min(len(jobs) + 1, os.cpu_count() or 1, 8))
        with concurrent.futures.ThreadPoolExecutor(max_workers=workers) as pool:
            futures = [pool.submit(_run, j, verbose) for j in jobs]
            module = None if missing else pool.submit(lambda: _run(calls_command(calls), verbose))
            for f in futures:
                f.result()
        _run([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", LIB_PATH + ".tmp"], verbose)
        os.replace(LIB_PATH + ".tmp", LIB_PATH)
        if os.path.exists(CALLS_PATH):
            os.remove(CALLS_PATH)          # never one of another build's
        if module is None:
            print(f"the module of the float operators' calls is left out: no {', '.join(missing)}", file=sys.stderr)
        else:
            module.result()
            shutil.copyfile(calls, CALLS_PATH + ".tmp")
            os.replace(CALLS_PATH + ".tmp", CALLS_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose=True))
