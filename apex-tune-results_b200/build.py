"""Builds libapex_attn.so in-tree (next to the apex_attn package) with nvcc for sm_100a, and then the
Python module _calls.so beside it with g++.

Usage: python apex-tune-results_b200/build.py [--verbose] [--force] [--strict]
Each source is compiled to an object under _build/ (side by side, and only when it or a
header changed), then linked. The library links the CUDA runtime statically and resolves
cuTensorMapEncodeTiled through cudaGetDriverEntryPoint, so it needs no -lcuda and loads on
a machine without a GPU; nvcc is all that it needs. _calls.so, a shorter way for the host
from Python to some of the library's calls, uses the headers of the installed torch and links to
its libraries. Where it cannot be built (no torch, no headers, no C++ compiler) the package does
without, so that is a warning, and an error with --strict only.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
OUT = os.path.join(HERE, "apex_attn", "libapex_attn.so")
SOURCES = [os.path.join(CSRC, "attn_fwd.cu"), os.path.join(CSRC, "paged.cu")]
API = os.path.join(ROOT, "include", "apex_attn.h")
# Headers each source includes (a change in one recompiles only the sources that list it).
_SHARED = [API, *(os.path.join(CSRC, f) for f in ("runtime.h", "sm100_ptx.cuh", "attn_fwd_kernel.cuh"))]
HEADERS = {
    SOURCES[0]: _SHARED + [os.path.join(CSRC, f) for f in ("attn_fwd_tile_kernel.cuh", "attn_bwd_kernel.cuh")],
    SOURCES[1]: _SHARED + [os.path.join(CSRC, f) for f in ("attn_paged_kernel.cuh", "kv_cache_kernels.cuh")],
}
CALLS_SOURCE = os.path.join(CSRC, "torch_calls.cpp")
CALLS_OUT = os.path.join(HERE, "apex_attn", "_calls.so")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo", "-Xptxas", "-v",
         "-Xcompiler", "-fPIC", "-I", os.path.join(ROOT, "include"), "-I", CSRC]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def object_of(source: str) -> str:
    return os.path.join(OBJ, os.path.splitext(os.path.basename(source))[0] + ".o")


def newer(target: str, inputs: list[str]) -> bool:
    return os.path.exists(target) and all(os.path.getmtime(f) <= os.path.getmtime(target) for f in inputs)


def stale_sources() -> list[str]:
    return [s for s in SOURCES if not newer(object_of(s), [s, *HEADERS[s], __file__])]


def up_to_date() -> bool:
    inputs = [f for s in SOURCES for f in (s, *HEADERS[s])] + [__file__]
    return newer(OUT, inputs)


def torch_dir() -> str:
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        raise RuntimeError("torch is not installed")
    return os.path.dirname(spec.origin)


def calls_key() -> str:
    """What _calls.so is compiled against: it uses the insides of torch's tensors and Python's objects, so
    it is only good for these very versions. Compiled in, and compared when it is loaded."""
    with open(os.path.join(torch_dir(), "version.py")) as f:
        version = re.search(r"^__version__\s*=\s*['\"]([^'\"]+)['\"]", f.read(), re.MULTILINE)
    if version is None:
        raise RuntimeError("the installed torch names no version")
    return f"torch {version.group(1)} {sysconfig.get_config_var('SOABI')}"


def cxx() -> str:
    return os.environ.get("CXX", "g++")


def calls_stamp() -> str:
    """The key and the compiler's version: with another of either the module is built anew."""
    proc = subprocess.run([cxx(), "--version"], capture_output=True, text=True)
    return f"{calls_key()}\n{cxx()}: {proc.stdout.splitlines()[0] if proc.stdout else ''}\n"


def cxx11_abi() -> int:
    """The C++ library ABI that the installed torch was compiled with."""
    import torch
    return int(torch.compiled_with_cxx11_abi())


def calls_command(out: str) -> list[str]:
    torch = torch_dir()
    include = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include"),
               os.path.join(ROOT, "include")]
    libs = ["torch_python", "torch", "torch_cpu", "torch_cuda", "c10", "c10_cuda"]
    return [cxx(), "-O2", f'-DAPEX_CALLS_KEY="{calls_key()}"', "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={cxx11_abi()}", *("-I" + p for p in include), "-o", out, CALLS_SOURCE,
            "-L" + os.path.join(torch, "lib"), *("-l" + name for name in libs)]


def build_calls(force: bool = False) -> str:
    stamp, at = calls_stamp(), os.path.join(OBJ, "_calls.stamp")
    same = False
    if os.path.exists(at):
        with open(at) as f:
            same = f.read() == stamp
    if force or not same or not newer(CALLS_OUT, [CALLS_SOURCE, API, __file__]):
        tmp = CALLS_OUT + ".tmp"
        proc = subprocess.run(calls_command(tmp), capture_output=True, text=True)
        if proc.returncode != 0:
            sys.stderr.write(proc.stdout + proc.stderr)
            raise RuntimeError("g++ failed building _calls.so")
        os.replace(tmp, CALLS_OUT)
        os.makedirs(OBJ, exist_ok=True)
        with open(at, "w") as f:
            f.write(stamp)
    return CALLS_OUT


def build(force: bool = False, verbose: bool = False, strict: bool = False) -> str:
    """Builds both; returns the library's path. Without _calls.so: RuntimeError if `strict`, else a warning."""
    build_library(force, verbose)
    try:
        build_calls(force)
    except (RuntimeError, ImportError, OSError) as e:
        if os.path.exists(CALLS_OUT):  # of other sources: it may not fit the library
            os.remove(CALLS_OUT)
        if strict:
            raise RuntimeError(f"_calls.so was not built: {e}") from e
        warnings.warn(f"_calls.so was not built ({e}): the paged cache's calls take the longer way through Python")
    return OUT


def build_library(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return OUT
    os.makedirs(OBJ, exist_ok=True)
    nvcc = nvcc_path()
    jobs = []
    for source in SOURCES if force else stale_sources():
        cmd = [nvcc, *FLAGS, "-c", "-o", object_of(source) + ".tmp", source]
        jobs.append((source, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = []
    for source, job in jobs:
        log = job.communicate()[0]
        if job.returncode != 0:
            sys.stderr.write(log)
            failed.append(os.path.basename(source))
            continue
        if verbose:
            sys.stdout.write(log)
        os.replace(object_of(source) + ".tmp", object_of(source))
    if failed:
        raise RuntimeError("nvcc failed building libapex_attn.so: " + ", ".join(failed))
    tmp = OUT + ".tmp"
    proc = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC",
                           "-o", tmp, *map(object_of, SOURCES)], capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError("nvcc failed linking libapex_attn.so")
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--strict", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose, strict=a.strict))
