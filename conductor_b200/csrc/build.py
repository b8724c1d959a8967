"""Build libconductor_b200.so in-tree with nvcc for sm_100a.

Replaces the reference's per-graph compile-and-link step
(conductor/compiler/jit_compiler.py:260-343 runs `choreo -c -fpic` then `gcc -shared`;
conductor/compiler/host_wrapper.py:270-295 runs `g++ -shared` on the generated wrapper)
with one ahead-of-time build of the fixed kernel-template library.

Usage: python -m conductor_b200.csrc.build [--force] [--verbose]
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

CSRC = Path(__file__).resolve().parent
LIB_NAME = "libconductor_b200.so"
LIB_PATH = CSRC / LIB_NAME
CALL_MODULE_SOURCE = "cdr_torch.cpp"               # CPython module, linked against torch (conductor_b200/ops.py)
CALL_MODULE_PATH = CSRC / "_cdr_torch.so"
CALL_MODULE_STAMP = CSRC / "_cdr_torch.stamp"      # what the module was built for

# file -> extra flags.  The elementwise and reduction templates must not contract
# a*b+c into an fma: eager rounds the product and the sum separately.
SOURCES = {
    "cdr_api.cu": [],
    "cdr_elementwise.cu": ["--fmad=false"],
    "cdr_jit.cu": [],
    "cdr_reduce.cu": ["--fmad=false"],
    "cdr_softmax.cu": ["--fmad=false"],
    "cdr_layernorm.cu": [],
    "cdr_copy.cu": [],
    "cdr_gemm.cu": [],
    "cdr_attention.cu": [],
    "cdr_cache_attention.cu": [],
    "cdr_tile_attention.cu": [],
}

COMMON = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xcompiler", "-fvisibility=hidden",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or "/usr/local/cuda/bin/nvcc"
    return cand if os.path.exists(cand) else "nvcc"


def _deps_mtime() -> float:
    paths = list(CSRC.glob("*.cuh")) + [CSRC.parent.parent / "include" / "conductor_b200.h"]
    return max(p.stat().st_mtime for p in paths if p.exists())


def _compile(src: str, flags: list[str], verbose: bool) -> Path:
    obj = CSRC / (Path(src).stem + ".o")
    cmd = [_nvcc(), *COMMON, *flags, "-c", str(CSRC / src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas")
        cmd.insert(2, "-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{res.stdout}\n{res.stderr}")
    if verbose:
        sys.stderr.write(res.stderr)
    return obj


def call_module_identity() -> str:
    """The torch and the Python whose class layouts the call module is compiled against."""
    import torch

    return f"torch {torch.__version__} {sysconfig.get_config_var('SOABI')}"


def build_call_module(force: bool = False) -> Path:
    """Compile the host side of direct calls against the installed torch; returns its path."""
    import torch

    src, identity = CSRC / CALL_MODULE_SOURCE, call_module_identity()
    newest = max(src.stat().st_mtime, (CSRC.parent.parent / "include" / "conductor_b200.h").stat().st_mtime)
    fits = CALL_MODULE_STAMP.exists() and CALL_MODULE_STAMP.read_text() == identity
    if not force and fits and CALL_MODULE_PATH.exists() and CALL_MODULE_PATH.stat().st_mtime >= newest:
        return CALL_MODULE_PATH
    root = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f'-DCDR_BUILT_FOR="{identity}"',
           f"-isystem{root}/include", f"-isystem{root}/include/torch/csrc/api/include",
           f"-isystem{sysconfig.get_paths()['include']}", f"-isystem{cuda}/include",
           str(src), "-o", str(CALL_MODULE_PATH), f"-L{root}/lib", "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    CALL_MODULE_STAMP.write_text(identity)
    return CALL_MODULE_PATH


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every kernel template, link the shared library and build the call module; returns the library's path.

    Without a C++ compiler or torch's headers the library stands alone: callers of the C ABI and compiled graphs need
    nothing else, and a direct operator call says what it misses."""
    with ThreadPoolExecutor(max_workers=1) as side:
        module = side.submit(build_call_module, force)
        path = build_library(force, verbose)
        try:
            module.result()
        except Exception as exc:
            warnings.warn(f"the call module of conductor_b200.ops was not built: {exc}", RuntimeWarning, stacklevel=2)
    return path


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile every kernel template and link the shared library; returns its path."""
    dep_time = _deps_mtime()
    todo = []
    for src, flags in SOURCES.items():
        obj = CSRC / (Path(src).stem + ".o")
        src_time = max((CSRC / src).stat().st_mtime, dep_time)
        if force or verbose or not obj.exists() or obj.stat().st_mtime < src_time:
            todo.append((src, flags))
    if todo:
        with ThreadPoolExecutor(max_workers=min(len(todo), os.cpu_count() or 1)) as pool:
            list(pool.map(lambda sf: _compile(sf[0], sf[1], verbose), todo))
    objs = [str(CSRC / (Path(s).stem + ".o")) for s in SOURCES]
    if todo or not LIB_PATH.exists():
        cmd = [_nvcc(), "-shared", "-o", str(LIB_PATH), *objs, "-cudart", "shared", "-ldl"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(path)
