"""Builds libfmoe_b200.so (sm_100a only) in-tree with nvcc, and the torch binding with g++."""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ_DIR = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libfmoe_b200.so")
SOURCES = ["sorting.cu", "rows.cu", "gemm.cu", "api.cu", "ep.cu", "router.cu", "silu.cu", "grouped.cu", "block_matmul.cu"]
HEADERS = ["ptx.cuh", "gemm.cuh", "gemm_block.cuh", "scales.cuh", "plan.hpp", "internal.h", "host.cuh", "grouped.cuh", "block_matmul.cuh", "block_small.cuh", "block_hw.cuh", os.path.join("..", "..", "include", "fused_moe_c.h")]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC,-fvisibility=hidden", "--expt-relaxed-constexpr"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    return "nvcc"


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def build(force: bool = False, verbose: bool = False, checked: bool = False, timing_switches: bool = False,
          wait_limit_switch: bool = False) -> str:
    """Builds the product library, or with checked=True libfmoe_b200_checked.so (the same
    sources with -DFMOE_BOUNDS_CHECKS), or with timing_switches=True libfmoe_b200_timing.so
    (-DFMOE_TIMING_SWITCHES: FMOE_DEBUG_FLAGS / FMOE_GEMM_MODE are honoured; results are invalid
    while they are set), or with wait_limit_switch=True libfmoe_b200_waits.so (-DFMOE_WAIT_LIMIT_SWITCH:
    fmoe_set_wait_limit sets how long a wait in a kernel may take).  The variants never replace the
    product library."""
    if checked or timing_switches:
        return _build_variant("checked" if checked else "timing",
                              ["-DFMOE_BOUNDS_CHECKS"] if checked else ["-DFMOE_TIMING_SWITCHES"], force, verbose)
    if wait_limit_switch:      # the operators' kernels; the rest is the product library's
        return _build_variant("waits", ["-DFMOE_WAIT_LIMIT_SWITCH"], force, verbose, only=("grouped.cu", "block_matmul.cu"))
    lib = _build_variant("", [], force, verbose)
    build_binding(force, verbose)
    return lib


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """Builds _fmoe_torch.so, the CPython binding of the operators in ops.py (host code only, g++ and
    torch's headers).  It does not link the library: ops.py passes it the entry points."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    src = os.path.join(CSRC, "torch_binding.cpp")
    out = os.path.join(HERE, "_fmoe_torch.so")
    made_for = os.path.join(OBJ_DIR, "_fmoe_torch.made_for")
    if not force and not _stale(out, [src, os.path.join(HERE, "..", "include", "fused_moe_c.h")]) and _recorded(made_for) == _binding_made_for():
        return out
    cuda = os.path.dirname(os.path.dirname(_nvcc())) if os.path.sep in _nvcc() else "/usr/local/cuda"
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-isystem{i}" for i in include], src, "-o", out,
           f"-L{torch_lib}", "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda", f"-Wl,-rpath,{torch_lib}"]
    env = {k: v for k, v in os.environ.items() if k not in ("CC", "CXX")}
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, env=env)
    if verbose or r.returncode != 0:
        print(" ".join(cmd))
        print(r.stdout)
    if r.returncode != 0:
        raise RuntimeError("g++ failed for torch_binding.cpp")
    os.makedirs(OBJ_DIR, exist_ok=True)
    with open(made_for, "w") as f:
        f.write(_binding_made_for())
    return out


def _binding_made_for() -> str:
    """What the binding is compiled against: it loads with no other torch or interpreter."""
    import torch

    return f"torch {torch.__version__}, {sys.implementation.cache_tag}"


def _recorded(path: str) -> str:
    try:
        with open(path) as f:
            return f.read()
    except OSError:
        return ""


def _build_variant(suffix: str, defines: list, force: bool, verbose: bool, only=tuple(SOURCES)) -> str:
    if set(only) != set(SOURCES):
        _build_variant("", [], force, verbose)
    product = globals()["OBJ_DIR"]
    OBJ_DIR = os.path.join(HERE, "build" + ("_" + suffix if suffix else ""))
    LIB = os.path.join(HERE, "libfmoe_b200" + ("_" + suffix if suffix else "") + ".so")
    NVCC_FLAGS = globals()["NVCC_FLAGS"] + defines
    os.makedirs(OBJ_DIR, exist_ok=True)
    hdrs = [os.path.join(CSRC, h) for h in HEADERS]
    jobs = []
    for src in only:
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ_DIR, src.replace(".cu", ".o"))
        if force or _stale(o, [s] + hdrs):
            jobs.append([_nvcc(), *NVCC_FLAGS, "-Xptxas", "-v", "-c", s, "-o", o])
    env = dict(os.environ)
    env.pop("CC", None)
    env.pop("CXX", None)

    def run(cmd):
        r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, env=env)
        return cmd, r.returncode, r.stdout

    with ThreadPoolExecutor(max_workers=4) as ex:
        for cmd, rc, out in ex.map(run, jobs):
            # ptxas -v output (registers, spills, shared memory per kernel) is kept beside the object
            with open(cmd[-1] + ".log", "w") as f:
                f.write(out)
            if verbose or rc != 0:
                print(" ".join(cmd))
                print(out)
            if rc != 0:
                raise RuntimeError(f"nvcc failed for {cmd[-3]}")
    objs = [os.path.join(OBJ_DIR if s in only else product, s.replace(".cu", ".o")) for s in SOURCES]
    if force or jobs or _stale(LIB, objs):
        cmd = [_nvcc(), "-shared", "-o", LIB, *objs, "-gencode", "arch=compute_100a,code=sm_100a"]
        r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, env=env)
        if r.returncode != 0:
            print(r.stdout)
            raise RuntimeError("link failed")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True, checked="--checked" in sys.argv,
                timing_switches="--timing-switches" in sys.argv))
