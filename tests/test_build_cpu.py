"""Which parts of the library a build makes anew, with a compiler that only writes down what it was asked for."""
import os
import stat

import pytest

from decode_matmul_b200 import build

NVCC = """#!/usr/bin/env python3
import sys
if "--version" in sys.argv:
    print("nvcc of the test, VERSION")
    sys.exit()
open("LOG", "a").write(" ".join(sys.argv[1:]) + "\\n")
open(sys.argv[sys.argv.index("-o") + 1], "w").write("made")
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A library of two units that share one header; returns (its folder, what was made since the last look)."""
    (tmp_path / "bin").mkdir()
    (tmp_path / "csrc").mkdir()
    (tmp_path / "include").mkdir()
    log = tmp_path / "log"

    def compiler(version):
        path = tmp_path / "bin" / "nvcc"
        path.write_text(NVCC.replace("VERSION", version).replace("LOG", str(log)))
        path.chmod(path.stat().st_mode | stat.S_IXUSR)

    compiler("1")
    for name, text in (("a.cu", '#include "both.h"\n'), ("b.cu", '#include "both.h"\n#include "b.h"\n'), ("both.h", ""), ("b.h", "")):
        (tmp_path / "csrc" / name).write_text(text)
    (tmp_path / "include" / "dmm.h").write_text("")
    monkeypatch.setenv("PATH", f"{tmp_path / 'bin'}:{os.environ['PATH']}")
    monkeypatch.setattr(build, "HERE", str(tmp_path / "csrc"))
    monkeypatch.setattr(build, "CSRC", str(tmp_path / "csrc"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "UNITS", ("a.cu", "b.cu"))

    def made():
        lines = log.read_text().splitlines() if log.exists() else []
        log.write_text("")
        return sorted(os.path.basename(line.split()[-1]) for line in lines if "-c" in line.split()), any("-shared" in line for line in lines)

    return tmp_path, made, compiler


def touch(tree, *names):
    """Makes files newer than everything else there is."""
    newest = max(os.path.getmtime(os.path.join(root, f)) for root, _, files in os.walk(tree) for f in files)
    for name in names:
        os.utime(tree / "csrc" / name, (newest + 10, newest + 10))


def test_only_what_has_changed_is_made_anew(tree):
    d, made, _ = tree
    build.build()
    assert made() == (["a.cu", "b.cu"], True)
    build.build()
    assert made() == ([], False)
    touch(d, "b.h")
    build.build()
    assert made() == (["b.cu"], True)


def test_objects_of_other_flags_or_another_compiler_are_not_linked(tree, monkeypatch):
    d, made, compiler = tree
    build.build()
    made()
    monkeypatch.setattr(build, "NVCC_FLAGS", [*build.NVCC_FLAGS, "-DOTHER"])
    touch(d, "b.h")
    build.build()
    assert made() == (["a.cu", "b.cu"], True)
    compiler("2")
    touch(d, "b.h")
    build.build()
    assert made() == (["a.cu", "b.cu"], True)


def test_an_object_of_unknown_origin_is_made_anew(tree):
    d, made, _ = tree
    for name in ("a.o", "b.o"):
        (d / "csrc" / name).write_text("from somewhere")
        touch(d, name)
    build.build()
    assert made() == (["a.cu", "b.cu"], True)
