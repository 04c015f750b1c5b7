"""Builds libtilegym_b200.so in-tree with nvcc for sm_100a.

    python -m tilegym_b200.build [--force] [--verbose]

One object per .cu file (compiled in parallel), linked into
tilegym_b200/libtilegym_b200.so with the CUDA runtime linked statically, so the
library has no dependency on torch or on a particular libcudart on the path.
Beside it tilegym_b200/_bind.so, a small torch extension (C++ only) that calls
the library for the decode-sized operators with less host time than ctypes.
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
OBJ_DIR = os.path.join(PKG_DIR, "build")
LIB_PATH = os.path.join(PKG_DIR, "libtilegym_b200.so")
BIND_PATH = os.path.join(PKG_DIR, "_bind.so")

SOURCES = ["api.cu", "gemm_pertensor.cu", "gemm_pertensor_2cta.cu", "gemm_blockscaled.cu", "gemm_blockscaled_wide.cu", "gemm_blockscaled_smallm.cu", "gemm_smallm.cu", "quant.cu", "group_quant.cu", "no_alloc.cu", "selftest.cu", "moe.cu", "rms_norm.cu", "kv_cache.cu",
           "attention.cu", "attention_few_rows.cu", "attention_many_rows.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; set NVCC or put it on PATH")
    return cand


def _newer(target: str, deps) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(d) <= t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    nvcc = _nvcc()
    os.makedirs(OBJ_DIR, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    headers.append(os.path.join(PKG_DIR, "..", "include", "tilegym_b200.h"))
    jobs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ_DIR, src.replace(".cu", ".o"))
        if force or not _newer(o, [s] + headers):
            extra = os.environ.get("TILEGYM_B200_NVCC_EXTRA", "").split()  # e.g. -DTG_TRACE for phase stamps
            cmd = [nvcc] + NVCC_FLAGS + extra + (["-Xptxas", "-v"] if verbose else []) + ["-c", s, "-o", o]
            jobs.append((src, cmd))
    if jobs:
        with cf.ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
            futs = {ex.submit(subprocess.run, cmd, capture_output=True, text=True): src for src, cmd in jobs}
            for f in cf.as_completed(futs):
                r = f.result()
                if verbose or r.returncode != 0:
                    sys.stderr.write(f"--- {futs[f]}\n{r.stdout}{r.stderr}")
                if r.returncode != 0:
                    raise RuntimeError(f"nvcc failed on {futs[f]}")
    objs = [os.path.join(OBJ_DIR, s.replace(".cu", ".o")) for s in SOURCES]
    if force or jobs or not _newer(LIB_PATH, objs):
        cmd = [nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB_PATH] + objs + ["-cudart", "static", "-ldl"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    try:
        build_bind(force)
    except Exception as e:  # g++, torch's headers: the library does without
        if os.path.exists(BIND_PATH):
            os.remove(BIND_PATH)  # of an older build, which may call the library otherwise
        sys.stderr.write(f"{e}: the library is built without the extension; decode-sized calls go through ctypes\n")
    return LIB_PATH


def build_bind(force: bool = False) -> str:
    import sysconfig

    import torch

    src = os.path.join(CSRC, "torch_bind.cpp")
    stamp = os.path.join(OBJ_DIR, "bind.torch")  # the version that it was built for
    if not force and _newer(BIND_PATH, [src, os.path.join(PKG_DIR, "..", "include", "tilegym_b200.h")]) and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == torch.__version__:
                return BIND_PATH

    root = os.path.dirname(os.path.abspath(torch.__file__))
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           f'-DTG_TORCH_VERSION="{torch.__version__}"',
           src, "-o", BIND_PATH] + [f"-I{p}" for p in include]
    cmd += [f"-L{os.path.join(root, 'lib')}", f"-L{PKG_DIR}", "-l:libtilegym_b200.so", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python",
            "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("g++ failed on torch_bind.cpp")
    with open(stamp, "w") as f:
        f.write(torch.__version__)
    return BIND_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
