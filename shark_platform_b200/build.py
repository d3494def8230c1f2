"""Builds the CUDA library in-tree: csrc/*.cu -> lib/libb200moe.so (sm_100a only), and the
torch binding of the cache operators: csrc/attention_ops.cpp -> lib/_attention_ops.so.

nvcc cross-compiles without a GPU.  Objects are rebuilt only when a source or
header is newer, the binding also when torch, Python or its command is another.  Run as `python -m shark_platform_b200.build [--force] [--verbose]`.
"""
from __future__ import annotations

import importlib.util
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libb200moe.so")
OPS = os.path.join(LIBDIR, "_attention_ops.so")
OPS_STAMP = os.path.join(OBJ, "attention_ops.stamp")  # what OPS was built with
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CXX = os.environ.get("CXX", "g++")
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
    "-I", INCLUDE,
]


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers_mtime():
    paths = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    paths += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    return max(os.path.getmtime(p) for p in paths)


def _ops_command() -> list[str]:
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(NVCC))
    return [CXX, "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall", f"-I{root}/include",
            f"-I{root}/include/torch/csrc/api/include", f"-I{sysconfig.get_paths()['include']}", f"-I{cuda}/include",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", os.path.join(CSRC, "attention_ops.cpp"),
            "-o", OPS, f"-L{root}/lib", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]


def _ops_stamp() -> str:
    import sysconfig

    import torch

    return "\n".join([torch.__version__, str(sysconfig.get_config_var("SOABI")), *_ops_command(), ""])


def _ops_stale(headers: float) -> bool:
    if not (os.path.exists(OPS) and os.path.exists(OPS_STAMP)):
        return True
    with open(OPS_STAMP) as f:
        if f.read() != _ops_stamp():
            return True
    return os.path.getmtime(OPS) < max(os.path.getmtime(os.path.join(CSRC, "attention_ops.cpp")), headers)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    hdr = _headers_mtime()
    jobs = []
    objs = []
    for src in _sources():
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ, src[:-3] + ".o")
        objs.append(o)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr):
            cmd = [NVCC, *FLAGS, "-c", s, "-o", o]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append(cmd)

    # without torch there is nothing to bind to: the C library alone
    ops = importlib.util.find_spec("torch") is not None and (force or _ops_stale(hdr))
    if ops:
        jobs.append(_ops_command())

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    if jobs:
        with ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            for cmd, r in ex.map(run, jobs):
                if verbose or r.returncode != 0:
                    sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr + "\n")
                if r.returncode != 0:
                    raise RuntimeError(f"{os.path.basename(cmd[0])} failed: {' '.join(cmd)}")
    if ops:
        with open(OPS_STAMP, "w") as f:
            f.write(_ops_stamp())
    if any(cmd[0] == NVCC for cmd in jobs) or not os.path.exists(LIB):
        cmd = [NVCC, "-shared", "-o", LIB, *objs, "-cudart", "static",
               "-gencode", "arch=compute_100a,code=sm_100a"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
