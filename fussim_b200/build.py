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

import functools
import hashlib
import os
import re
import shutil
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


def _compile(job, verbose):
    """Runs a compile command into a file of its own, which takes the object's place when it is
    whole: a build that is killed, or another one beside it, leaves no half of an object."""
    cmd, target = job
    part = f"{target}.{os.getpid()}.part"
    try:
        res = _run([*cmd, "-o", part], verbose)
        os.replace(part, target)
        return res.stderr
    finally:
        if os.path.exists(part):
            os.remove(part)


def _compile_all(jobs, verbose):
    """Run the compile jobs, (command, object), side by side; returns what each wrote to standard
    error."""
    os.makedirs(OBJ, exist_ok=True)
    with ThreadPoolExecutor(max_workers=max(1, os.cpu_count() or 1)) as pool:
        return list(pool.map(lambda job: _compile(job, verbose), jobs))


@functools.lru_cache(maxsize=None)
def _compiler_version(compiler):
    return _run([compiler, "--version"], False).stdout


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


def _object(source, command, *versions):
    """The object file of a source compiled by this command (all but the output): its name tells
    the command, the compiler's version and the others given, so that an object is used again only
    for what it was compiled with. Where the tree lies does not count."""
    key = "\0".join([*command, _compiler_version(command[0]), *versions]).replace(ROOT, "")
    key = hashlib.sha256(key.encode()).hexdigest()[:12]
    return os.path.join(OBJ, f"{os.path.basename(source)}.{key}.o")


def _link(cmd, target, verbose):
    part = f"{target}.{os.getpid()}.part"
    try:
        _run([*cmd, "-o", part], verbose)
        os.replace(part, target)
    finally:
        if os.path.exists(part):
            os.remove(part)


def _forget_others(sources, objects):
    """Removes the objects of these sources that other commands compiled."""
    for name in os.listdir(OBJ):
        path = os.path.join(OBJ, name)
        if name.endswith(".o") and path not in objects and \
                any(name.startswith(os.path.basename(s) + ".") for s in sources):
            os.remove(path)


def build_engine(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    cus = [s for s in engine_sources() if s.endswith(".cu")]
    if not force and shutil.which(_nvcc()) is None and \
            not _stale(LIB, [*engine_sources(), os.path.join(INCLUDE, "fussim_b200.h")]):
        return LIB  # built elsewhere
    commands = {cu: [_nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, "-I", INCLUDE, "-c", cu] for cu in cus}
    objects = {cu: _object(cu, commands[cu]) for cu in cus}
    jobs = [([*commands[cu], *(["-Xptxas=-v"] if ptxas_info else [])], objects[cu]) for cu in cus
            if force or ptxas_info or _stale(objects[cu], _includes(cu))]
    if not jobs and not _stale(LIB, objects.values()):
        return LIB
    infos = _compile_all(jobs, verbose)
    _link([_nvcc(), *ARCH_FLAGS, "-shared", *objects.values()], LIB, verbose)
    _forget_others(cus, objects.values())
    if ptxas_info:
        sys.stdout.write("".join(infos))
    return LIB


def build_torch_ext(force: bool = False, verbose: bool = False) -> str:
    # The extension links the library by name and finds it at run time, so a rebuilt
    # library does not require relinking the extension.
    import torch
    from torch.utils import cpp_extension as ce

    cpps = [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith(".cpp")]
    incs = ce.include_paths(device_type="cuda") + [sysconfig.get_paths()["include"], INCLUDE]
    libdirs = ce.library_paths(device_type="cuda")
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    flags = ["g++", "-O3", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
             "-DTORCH_EXTENSION_NAME=_C", "-DTORCH_API_INCLUDE_EXTENSION_H",
             *[f"-I{i}" for i in incs]]
    if not force and shutil.which("g++") is None and \
            not _stale(EXT, {d for cpp in cpps for d in _includes(cpp)}):
        return EXT
    commands = {cpp: [*flags, "-c", cpp] for cpp in cpps}
    objects = {cpp: _object(cpp, commands[cpp], torch.__version__, sys.version) for cpp in cpps}
    jobs = [(commands[cpp], objects[cpp]) for cpp in cpps if force or _stale(objects[cpp], _includes(cpp))]
    if not jobs and not _stale(EXT, objects.values()):
        return EXT
    _compile_all(jobs, verbose)
    _link(["g++", "-shared", *objects.values(), *[f"-L{d}" for d in libdirs], f"-L{PKG}",
           "-lfussim_b200", "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10_cuda",
           "-ltorch_cuda", "-lcudart", "-Wl,-rpath,$ORIGIN"], EXT, verbose)
    _forget_others(cpps, objects.values())
    return EXT


def build_all(force: bool = False, verbose: bool = False) -> None:
    build_engine(force=force, verbose=verbose)
    build_torch_ext(force=force, verbose=verbose)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv, verbose=True)
    print(LIB)
    print(EXT)
