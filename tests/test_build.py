"""The library's build: what it compiles again, with a stand-in for the compiler."""
import os
import stat

import pytest


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source tree of two files, a compiler that notes its arguments and writes its output: (the build, what was compiled)."""
    from super_resolution_amd import _lib
    pkg = tmp_path / "pkg"
    for d in (pkg / "csrc", tmp_path / "include"):
        d.mkdir(parents=True)
    for f in (pkg / "csrc" / "a.hip", pkg / "csrc" / "b.hip", pkg / "csrc" / "c.hpp", tmp_path / "include" / "gpsr.h"):
        f.write_text("")
        os.utime(f, (1, 1))
    log, cc = tmp_path / "log", tmp_path / "cc"
    cc.write_text(f'#!/bin/bash\necho "$@" >> {log}\nwhile [ "$1" != -o ]; do shift; done\ntouch "$2"\n')
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    for name, value in (("_HERE", str(pkg)), ("_CSRC", str(pkg / "csrc")), ("LIB_PATH", str(pkg / "libgpsr.so")), ("HIPCC", str(cc))):
        monkeypatch.setattr(_lib, name, value)

    def build(**kw):
        log.write_text("")
        assert _lib.build(**kw) == str(pkg / "libgpsr.so") and (pkg / "libgpsr.so").exists()
        lines = log.read_text().splitlines()
        return sorted(os.path.basename(x.split()[-1]) for x in lines if " -c " in x), lines
    return build, pkg, _lib


def test_only_what_changed_is_compiled_again(tree):
    build, pkg, _ = tree
    assert build()[0] == ["a.hip", "b.hip"]
    assert build() == ([], [])
    later = os.stat(pkg / "libgpsr.so").st_mtime + 10
    os.utime(pkg / "csrc" / "b.hip", (later, later))
    assert build()[0] == ["b.hip"]
    assert build(force=True)[0] == ["a.hip", "b.hip"]


def test_other_flags_compile_everything_again(tree, monkeypatch):
    build, pkg, lib = tree
    build()
    monkeypatch.setattr(lib, "HIPCC_FLAGS", lib.HIPCC_FLAGS + ["-DOTHER"])
    compiled, lines = build()
    assert compiled == ["a.hip", "b.hip"] and all("-DOTHER" in x for x in lines if " -c " in x)
    assert build() == ([], [])
    os.remove(pkg / "build" / "command")      # objects of a build that did not say how
    assert build()[0] == ["a.hip", "b.hip"]
