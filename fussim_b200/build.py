"""In-tree build of the engine for sm_100a.

Produces, next to this file:

* ``libfussim_b200.so``  the C-ABI library (nvcc, no torch), declared in
  ``include/fussim_b200.h``;
* ``_C.so``              the thin torch extension over that library (g++ against torch's
  headers, rpath ``$ORIGIN`` so it finds the library beside it).

Run ``python -m fussim_b200.build`` (or ``__graft_entry__.build()``). Nothing is cached
outside the repository, so the built files travel with a copy of the tree.
"""

from __future__ import annotations

import os
import re
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB = os.path.join(PKG, "libfussim_b200.so")
EXT = os.path.join(PKG, "_C.so")
OBJ = os.path.join(PKG, "_build")  # object files, one per source, kept between builds

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3"]


def _nvcc() -> str:
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    path = os.path.join(home, "bin", "nvcc")
    return path if os.path.exists(path) else "nvcc"


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"build step failed: {cmd[0]} (exit {res.returncode})")
    return res


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def engine_sources():
    return [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC))
            if f.endswith((".cu", ".cuh", ".h"))]


def _compile_all(commands, verbose):
    """Run the compile commands side by side; returns what each wrote to standard error."""
    os.makedirs(OBJ, exist_ok=True)
    with ThreadPoolExecutor(max_workers=max(1, os.cpu_count() or 1)) as pool:
        return [r.stderr for r in pool.map(lambda cmd: _run(cmd, verbose), commands)]


def _includes(source, seen=None):
    """The source and the headers of csrc/ and include/ that it includes, directly or not."""
    seen = {} if seen is None else seen
    if source in seen:
        return list(seen)
    seen[source] = True
    with open(source) as f:
        names = re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M)
    for name in names:
        for folder in (CSRC, INCLUDE):
            path = os.path.join(folder, name)
            if os.path.exists(path):
                _includes(path, seen)
    return list(seen)


def _object(source):
    return os.path.join(OBJ, os.path.basename(source) + ".o")


def build_engine(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    deps = engine_sources() + [os.path.join(INCLUDE, "fussim_b200.h")]
    if not force and not _stale(LIB, deps):
        return LIB
    cus = [s for s in engine_sources() if s.endswith(".cu")]
    jobs = []
    for cu in cus:
        if force or ptxas_info or _stale(_object(cu), _includes(cu)):
            cmd = [_nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, "-c", "-I", INCLUDE, "-o", _object(cu), cu]
            if ptxas_info:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append(cmd)
    infos = _compile_all(jobs, verbose)
    _run([_nvcc(), *ARCH_FLAGS, "-shared", "-o", LIB, *[_object(cu) for cu in cus]], verbose)
    if ptxas_info:
        sys.stdout.write("".join(infos))
    return LIB


def build_torch_ext(force: bool = False, verbose: bool = False) -> str:
    # The extension links the library by name and finds it at run time, so a rebuilt
    # library does not require relinking the extension.
    cpps = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith(".cpp")]
    deps = sorted({d for cpp in cpps for d in _includes(cpp)})
    if not force and not _stale(EXT, deps):
        return EXT
    import torch
    from torch.utils import cpp_extension as ce

    incs = ce.include_paths(device_type="cuda") + [sysconfig.get_paths()["include"], INCLUDE]
    libdirs = ce.library_paths(device_type="cuda")
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    flags = ["-O3", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
             "-DTORCH_EXTENSION_NAME=_C", "-DTORCH_API_INCLUDE_EXTENSION_H",
             *[f"-I{i}" for i in incs]]
    _compile_all([["g++", *flags, "-c", cpp, "-o", _object(cpp)] for cpp in cpps
                  if force or _stale(_object(cpp), _includes(cpp))], verbose)
    cmd = ["g++", "-shared", *[_object(cpp) for cpp in cpps], "-o", EXT,
           *[f"-L{d}" for d in libdirs], f"-L{PKG}", "-lfussim_b200", "-lc10", "-ltorch",
           "-ltorch_cpu", "-ltorch_python", "-lc10_cuda", "-ltorch_cuda", "-lcudart",
           "-Wl,-rpath,$ORIGIN"]
    _run(cmd, verbose)
    return EXT


def build_all(force: bool = False, verbose: bool = False) -> None:
    build_engine(force=force, verbose=verbose)
    build_torch_ext(force=force, verbose=verbose)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv, verbose=True)
    print(LIB)
    print(EXT)
