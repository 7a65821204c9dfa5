"""ps_amd.build's rule of what is compiled again, with a stand-in for hipcc that writes what it was asked to write."""
import os
import stat

import pytest


@pytest.fixture
def tree(tmp_path, monkeypatch):
    from ps_amd import build as b
    csrc, inc = tmp_path / "ps_amd" / "csrc", tmp_path / "include"
    csrc.mkdir(parents=True)
    inc.mkdir()
    for f in ("a.hip", "b.hip"):
        (csrc / f).write_text("// nothing\n")
    (csrc / "h.h").write_text("\n")
    log = tmp_path / "log"
    cc = tmp_path / "hipcc"
    cc.write_text('#!/bin/sh\necho "$@" >> %s\nwhile [ "$1" != -o ]; do shift; done\necho built > "$2"\n' % log)
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    for k, v in (("HERE", tmp_path / "ps_amd"), ("CSRC", csrc), ("OBJ", tmp_path / "obj"), ("LIBDIR", tmp_path / "lib"), ("LIB", tmp_path / "lib" / "x.so")):
        monkeypatch.setattr(b, k, str(v))
    monkeypatch.setattr(b, "SOURCES", ["a.hip", "b.hip"])
    monkeypatch.setenv("HIPCC", str(cc))
    monkeypatch.delenv("PS_AMD_EXTRA_FLAGS", raising=False)
    now = os.path.getmtime(csrc / "a.hip")
    for f in (csrc / "a.hip", csrc / "b.hip", csrc / "h.h"):
        os.utime(f, (now - 100, now - 100))

    def compiled():
        """the units compiled and the links made since the last call"""
        lines = log.read_text().splitlines() if log.exists() else []
        if log.exists():
            log.unlink()
        return sorted(os.path.basename(w) for ln in lines for w in ln.split() if w.endswith(".hip")), sum("-shared" in ln for ln in lines)
    return b, csrc, compiled, monkeypatch


def test_nothing_is_compiled_twice(tree):
    b, _, compiled, _ = tree
    b.build()
    assert compiled() == (["a.hip", "b.hip"], 1)
    b.build()
    assert compiled() == ([], 0)
    b.build(force=True)
    assert compiled() == (["a.hip", "b.hip"], 1)


def test_a_changed_source_or_header_is_compiled(tree):
    b, csrc, compiled, _ = tree
    b.build()
    compiled()
    later = os.path.getmtime(os.path.join(b.OBJ, "a.o")) + 10
    os.utime(csrc / "a.hip", (later, later))
    b.build()
    assert compiled()[0] == ["a.hip"]


def test_changed_flags_reach_every_unit(tree):
    """objects of another command line are not linked with new ones (a unit kept packed f32 instructions after they were switched off)"""
    b, _, compiled, mp = tree
    b.build()
    compiled()
    mp.setattr(b, "FLAGS", b.FLAGS + ["-DOTHER"])
    b.build()
    assert compiled() == (["a.hip", "b.hip"], 1)
    b.build()
    assert compiled() == ([], 0)
    mp.setenv("PS_AMD_EXTRA_FLAGS", "-DMORE")
    b.build()
    assert compiled() == (["a.hip", "b.hip"], 1)
    os.unlink(os.path.join(b.OBJ, "b.o.flags"))              # an object of unknown flags (a tree built before they were recorded)
    b.build()
    assert compiled() == (["b.hip"], 1)
