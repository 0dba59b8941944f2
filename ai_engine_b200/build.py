"""In-tree build of the CUDA library ``ai_engine_b200/libaie_conv.so``.

Translation units, compiled for sm_100a only and side by side: the conv path
(``csrc/aie_conv.cu``, which includes the ``k_*.cuh`` kernels), the sequence
operators (``csrc/aie_seq.cu``, the ``seq_*.cuh`` kernels) and, for the time they
take, the one-token kernels over states and the 4-bit cache
(``csrc/aie_read*.cu``).  Beside
it ``_seqcall.so``, the sequence operators' binding on torch tensors
(``csrc/seq_bind.cpp``), which is linked against it; where torch or Python's
headers are missing it is left out, with a message (the C ABI needs neither).
The CUDA runtime is linked statically, so the library depends on nothing but
the driver; the tensor-map encoder is fetched from the driver at run time.

    python ai_engine_b200/build.py [-v] [--changed]     # needs nvcc alone
"""
from __future__ import annotations

import glob
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libaie_conv.so")
UNITS = ("aie_conv", "aie_seq", "aie_read16", "aie_read4_f16", "aie_read4_bf16")
OBJ = os.path.join(HERE, "_build")
BIND = os.path.join(HERE, "_seqcall.so")
BIND_SRC = os.path.join(CSRC, "seq_bind.cpp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-fvisibility=hidden",
    "-cudart", "static",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources(unit=None):
    """The files a translation unit is made from (None: all of them)."""
    if unit is None:
        return sorted({f for u in UNITS for f in sources(u)})
    headers = [f for f in glob.glob(os.path.join(CSRC, "*.cuh"))
               if not os.path.basename(f).startswith("seq_" if unit == "aie_conv" else "k_")]
    api = ["aie_conv.h"] if unit == "aie_conv" else ["aie_conv.h", "aie_seq.h"]
    return [os.path.join(CSRC, unit + ".cu"), *headers, *(os.path.join(ROOT, "include", h) for h in api)]


def _older(path, files) -> bool:
    return not os.path.exists(path) or any(os.path.getmtime(f) > os.path.getmtime(path) for f in files)


def stale() -> bool:
    return _older(LIB, sources()) or _older(BIND, _bind_sources())


def _bind_sources():
    return [BIND_SRC, *(os.path.join(ROOT, "include", h) for h in ("aie_conv.h", "aie_seq.h"))]


def bind_needs() -> str:
    """What the binding needs and this machine lacks."""
    if importlib.util.find_spec("torch") is None:
        return "torch"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python's headers"
    return ""


def _bind_command(out: str):
    import torch
    from torch.utils import cpp_extension
    inc = [f for d in (sysconfig.get_paths()["include"], *cpp_extension.include_paths("cuda")) for f in ("-isystem", d)]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *inc, BIND_SRC, "-o", out,
            "-L", libs, "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-L", HERE, "-l:libaie_conv.so",
            "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = False, extra=()) -> str:
    if not force and not stale():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    objs, jobs, tmp = [], [], f".tmp{os.getpid()}"
    for u in UNITS:
        obj = os.path.join(OBJ, u + ".o")
        objs.append(obj)
        if force or _older(obj, sources(u)):
            cmd = [nvcc(), *NVCC_FLAGS, *extra, "-c", os.path.join(CSRC, u + ".cu"), "-o", obj + tmp]
            if verbose:
                print(" ".join(cmd), flush=True)
            jobs.append((obj, cmd, subprocess.Popen(cmd)))
    for obj, cmd, p in jobs:
        if p.wait() == 0:
            os.replace(obj + tmp, obj)
    for _, cmd, p in jobs:
        if p.returncode:
            raise subprocess.CalledProcessError(p.returncode, cmd)
    if jobs or _older(LIB, objs):
        subprocess.run([nvcc(), *NVCC_FLAGS, "-shared", *objs, "-o", LIB + tmp], check=True)
        os.replace(LIB + tmp, LIB)
    if force or _older(BIND, _bind_sources()):
        lacks = bind_needs()
        if lacks:
            print(f"{BIND} is left out: {lacks} not found", file=sys.stderr)
        else:
            subprocess.run(_bind_command(BIND + tmp), check=True)
            os.replace(BIND + tmp, BIND)
    return LIB


if __name__ == "__main__":
    extra = ["-Xptxas", "-v"] if "-v" in sys.argv else []
    print(build(force="--changed" not in sys.argv, verbose=True, extra=extra))
