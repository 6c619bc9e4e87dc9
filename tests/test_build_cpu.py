"""Which objects a build uses again (runs without a GPU; a stand-in compiler writes down its command)."""

import os
import stat
import sys

import pytest

from fussim_b200 import build

COMPILER = """#!{python}
import os, sys, time
args = sys.argv[1:]
if args == ["--version"]:
    print(open({folder!r} + "/version").read())
    raise SystemExit
out = args[args.index("-o") + 1]
with open({folder!r} + "/log", "a") as log:
    log.write(("link " if "-shared" in args else "compile ") + " ".join(a for a in args if a.endswith((".cu", ".cpp"))) + "\\n")
with open(out, "w") as f:
    f.write("half")
    f.flush()
    if os.path.exists({folder!r} + "/fail"):
        raise SystemExit(1)
    f.write(" ".join(args))
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A tree of two sources and a header, and a compiler."""
    root = tmp_path / "tree"
    csrc, include = root / "pkg" / "csrc", root / "include"
    csrc.mkdir(parents=True)
    include.mkdir()
    (include / "fussim_b200.h").write_text("")
    (csrc / "a.cu").write_text('#include "fussim_b200.h"\n#include "a.cuh"\n')
    (csrc / "a.cuh").write_text("")
    (csrc / "b.cu").write_text("")
    (tmp_path / "version").write_text("1.0")
    compiler = tmp_path / "nvcc"
    compiler.write_text(COMPILER.format(python=sys.executable, folder=str(tmp_path)))
    compiler.chmod(compiler.stat().st_mode | stat.S_IXUSR)
    for name, value in (("ROOT", root), ("PKG", root / "pkg"), ("CSRC", csrc), ("INCLUDE", include),
                        ("LIB", root / "pkg" / "lib.so"), ("OBJ", root / "pkg" / "_build")):
        monkeypatch.setattr(build, name, str(value))
    monkeypatch.setattr(build, "_nvcc", lambda: str(compiler))
    new_process()
    yield tmp_path
    new_process()


def new_process():
    """What a process keeps of the compiler is forgotten."""
    build._compiler_version.cache_clear()


def objects():
    return {name: open(os.path.join(build.OBJ, name)).read() for name in os.listdir(build.OBJ)}


def steps(tree):
    """What the compiler has been asked for since the last look."""
    log = tree / "log"
    text = log.read_text() if log.exists() else ""
    log.write_text("")
    return sorted(os.path.basename(line.split(" ", 1)[-1]) or "link" for line in text.splitlines())


def age(path, seconds):
    t = os.path.getmtime(path) - seconds
    os.utime(path, (t, t))


def test_only_what_changed(tree):
    build.build_engine()
    assert steps(tree) == ["a.cu", "b.cu", "link"]
    build.build_engine()
    assert steps(tree) == []
    for name in objects():
        age(os.path.join(build.OBJ, name), 100)
    age(build.LIB, 50)
    for name in ("a.cu", "b.cu", "a.cuh"):
        age(os.path.join(build.CSRC, name), 200)
    age(os.path.join(build.INCLUDE, "fussim_b200.h"), 200)
    build.build_engine()
    assert steps(tree) == []
    os.utime(os.path.join(build.CSRC, "a.cuh"))
    build.build_engine()
    assert steps(tree) == ["a.cu", "link"]
    build.build_engine(force=True)
    assert steps(tree) == ["a.cu", "b.cu", "link"]


def test_other_flags_and_another_compiler(tree, monkeypatch):
    build.build_engine()
    steps(tree)
    monkeypatch.setattr(build, "NVCC_FLAGS", [*build.NVCC_FLAGS, "--fmad=false"])
    build.build_engine()
    assert steps(tree) == ["a.cu", "b.cu", "link"]
    assert all("--fmad=false" in text for text in objects().values())
    (tree / "version").write_text("1.1")
    new_process()
    build.build_engine()
    assert steps(tree) == ["a.cu", "b.cu", "link"]
    assert len(objects()) == 2  # the old ones are gone


def test_a_tree_that_moved(tree, monkeypatch):
    build.build_engine()
    steps(tree)
    os.rename(tree / "tree", tree / "moved")
    for name in ("PKG", "CSRC", "INCLUDE", "LIB", "OBJ", "ROOT"):
        monkeypatch.setattr(build, name, getattr(build, name).replace(str(tree / "tree"), str(tree / "moved")))
    build.build_engine()
    assert steps(tree) == []


def test_a_compiler_that_fails_leaves_nothing(tree, capfd):
    build.build_engine()
    steps(tree)
    before, lib = objects(), open(build.LIB).read()
    (tree / "fail").write_text("")
    with pytest.raises(RuntimeError, match="build step failed"):
        build.build_engine(force=True)
    assert objects() == before and open(build.LIB).read() == lib
    assert sorted(os.listdir(build.PKG)) == ["_build", "csrc", "lib.so"]


def test_without_a_compiler(tree, monkeypatch):
    build.build_engine()
    monkeypatch.setattr(build, "_nvcc", lambda: str(tree / "none"))
    new_process()
    assert build.build_engine() == build.LIB
    os.utime(os.path.join(build.CSRC, "b.cu"), (2e9, 2e9))
    with pytest.raises(OSError):
        build.build_engine()
