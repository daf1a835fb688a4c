"""In-tree build of the C-ABI CUDA library (libpsa_b200.so) for sm_100a.

    python pyramid-sparse-attention_b200/build.py [--force] [-v]

Each csrc/*.cu is compiled to build/*.o in parallel with
``nvcc -gencode arch=compute_100a,code=sm_100a -lineinfo -O3`` and linked into
psa_b200/libpsa_b200.so; csrc/calls.cpp, the Python entry to some of its calls, is compiled with the host compiler
against torch's headers and linked with that library into a module whose name says which torch and which Python it is for
(calls_name.py).  Objects are reused when they are newer than every source and header.
"""
from __future__ import annotations

import glob
import importlib.util
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "psa_b200", "libpsa_b200.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CXX = os.environ.get("CXX", "g++")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "-Xcompiler", "-fPIC", "-Xptxas", "-v"]


def _newest_header() -> float:
    hdrs = glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        glob.glob(os.path.join(CSRC, "*.inl")) + glob.glob(os.path.join(HERE, "..", "include", "*.h"))
    return max(os.path.getmtime(h) for h in hdrs)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdr_t = _newest_header()
    jobs = []
    for s in srcs:
        o = os.path.join(OBJ, os.path.basename(s)[:-3] + ".o")
        stale = force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr_t)
        jobs.append((s, o, stale))

    def compile_one(job):
        s, o, stale = job
        if not stale:
            return o, ""
        r = subprocess.run([NVCC, *FLAGS, "-c", s, "-o", o], capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {s}:\n{r.stdout}\n{r.stderr}")
        return o, r.stderr

    with ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
        results = list(ex.map(compile_one, jobs))
    if verbose:
        for o, log in results:
            if log:
                print(f"== {os.path.basename(o)}\n{log}")
    objs = [o for o, _ in results]
    relink = force or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs)
    if relink:
        r = subprocess.run([NVCC, "-shared", "-o", LIB, *objs], capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    build_calls(force, hdr_t)
    return LIB


def calls_path() -> str:
    spec = importlib.util.spec_from_file_location("calls_name", os.path.join(HERE, "psa_b200", "calls_name.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return os.path.join(HERE, "psa_b200", mod.calls_name())


def build_calls(force: bool, hdr_t: float) -> None:
    try:
        import torch
    except ImportError:
        print("no torch: the C library alone")
        return
    src, out = os.path.join(CSRC, "calls.cpp"), calls_path()
    for old in glob.glob(os.path.join(HERE, "psa_b200", "_calls*.so")):
        if old != out:
            os.remove(old)       # of another torch or Python
    if not force and os.path.exists(out) and os.path.getmtime(out) >= max(os.path.getmtime(src), hdr_t):
        return
    at = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(NVCC)) or "/usr/local/cuda"
    include = [os.path.join(HERE, "..", "include"), os.path.join(at, "include"), os.path.join(at, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    abi = f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"
    r = subprocess.run([CXX, "-O2", "-std=c++17", "-fPIC", "-shared", abi, *[f"-I{i}" for i in include], src, "-o", out,
                        f"-L{os.path.dirname(LIB)}", f"-l:{os.path.basename(LIB)}", "-Wl,-rpath,$ORIGIN", f"-L{os.path.join(at, 'lib')}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"],
                       capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{CXX} failed on {src}:\n{r.stdout}\n{r.stderr}")


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
