"""Build recipe: compiles csrc/*.cu for sm_100a into lib/libstreamk_b200.so.

The library is a plain C-ABI shared object (no torch, no pybind): nvcc only, and build() needs
nothing else.  Objects are rebuilt when a source or header is newer than the object.  Beside it,
where torch is installed, the host compiler makes lib/sk_torch_host.<torch>-<python>.so from
csrc/host/sk_torch_host.cpp (build_host()), a small CPython module over torch's headers: the
shortcut from tensors to the C ABI that ops.py takes in plain cases.

STREAMK_B200_TRACE=1 builds a second library, lib/libstreamk_b200_trace.so, compiled with
-DSK_TRACE: its kernels record per-CTA timestamps while sk_debug_set_trace() names a buffer.
The ordinary library carries no tracing code.
"""
from __future__ import annotations

import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
OBJDIR = os.path.join(HERE, "build")
LIBNAME = "libstreamk_b200.so"
TRACE_LIBNAME = "libstreamk_b200_trace.so"
HOST_SRC = os.path.join(CSRC, "host", "sk_torch_host.cpp")
HOST_LIB = os.path.join(LIBDIR, "sk_torch_host.so")   # (see host_lib())
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def trace_build() -> bool:
    return os.environ.get("STREAMK_B200_TRACE") == "1"


def lib_path() -> str:
    return os.path.join(LIBDIR, TRACE_LIBNAME if trace_build() else LIBNAME)


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put it on PATH")


def _sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers() -> list[str]:
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh", ".inc"))]
    hs.append(os.path.join(HERE, "..", "include", "streamk_b200.h"))
    return hs


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _make(cmd: list[str], out: str) -> subprocess.CompletedProcess:
    """Runs a compiler or linker that writes `out`, under another name until it is whole: processes
    that find it missing at the same time, or load it meanwhile, never meet half a file."""
    part = f"{out}.{os.getpid()}.tmp"
    try:
        r = subprocess.run([*cmd, "-o", part], capture_output=True, text=True)
        if r.returncode == 0:
            os.replace(part, out)
    finally:
        if os.path.exists(part):
            os.remove(part)
    return r


def host_lib() -> str:
    """Path of the host module.  It is compiled against the insides of one torch and one Python, so its
    name tells which: another version of either has a file of its own instead of loading this one."""
    import torch
    tag = re.sub(r"[^\w.+-]", "_", f"torch{torch.__version__}-{sys.implementation.cache_tag}")
    return f"{HOST_LIB[:-len('.so')]}.{tag}.so"


def build_host(force: bool = False, verbose: bool = False) -> str:
    """Compile (if needed) the CPython module of the host fast path and return its path."""
    import torch
    header = os.path.join(HERE, "..", "include", "streamk_b200.h")
    out = host_lib()
    if not force and not _stale(out, [HOST_SRC, header]):
        return out
    os.makedirs(LIBDIR, exist_ok=True)
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    cxx = os.environ.get("CXX") or shutil.which("g++") or shutil.which("c++")
    if not cxx:
        raise RuntimeError("no C++ compiler found; set CXX")
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-I{d}" for d in (os.path.join(root, "include"),
                                os.path.join(root, "include", "torch", "csrc", "api", "include"),
                                sysconfig.get_paths()["include"], os.path.join(cuda, "include"))),
           HOST_SRC, f"-L{os.path.join(root, 'lib')}",
           "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    r = _make(cmd, out)
    if verbose or r.returncode != 0:
        sys.stderr.write(f"--- {os.path.basename(HOST_SRC)}\n{r.stdout}{r.stderr}\n")
    if r.returncode != 0:
        raise RuntimeError(f"compiling {HOST_SRC} failed")
    return out


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile (if needed) and return the path of the shared library, and where torch is installed the
    host module as well; without torch, or if the module does not compile, the library is all."""
    out = build_library(force, verbose)
    if importlib.util.find_spec("torch") is not None:
        try:
            build_host(force, verbose)
        except (ImportError, OSError, RuntimeError) as e:
            sys.stderr.write(f"{os.path.basename(HOST_SRC)} was not built: {e}\n")
    return out


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile (if needed) and return the path of the shared library."""
    objdir = OBJDIR + ("_trace" if trace_build() else "")
    os.makedirs(LIBDIR, exist_ok=True)
    os.makedirs(objdir, exist_ok=True)
    nvcc = _nvcc()
    headers = _headers()
    common = [nvcc, "-O3", "-std=c++17", "-lineinfo", *ARCH_FLAGS, "-Xcompiler", "-fPIC",
              "-Xptxas", "-v"]
    if trace_build():
        common.append("-DSK_TRACE")
    jobs = []
    objs = []
    for src in _sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src, *headers]):
            jobs.append((src, obj))

    def compile_one(job):
        src, obj = job
        return src, _make([*common, "-c", src], obj)

    with ThreadPoolExecutor(max_workers=max(1, min(8, len(jobs) or 1))) as ex:
        for src, r in ex.map(compile_one, jobs):
            if verbose or r.returncode != 0:
                sys.stderr.write(f"--- {os.path.basename(src)}\n{r.stdout}{r.stderr}\n")
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src}")
    out = lib_path()
    if force or jobs or _stale(out, objs):
        r = _make([nvcc, "-shared", *ARCH_FLAGS, *objs], out)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
