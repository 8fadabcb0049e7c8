"""CPU: the build recipe - what is compiled again, and with which flags (a recording stand-in for the compiler)."""
import os
import stat

import pytest

from pivotcvae_amd import build as b

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """two sources and a header under tmp_path; -> a function that builds and returns what the compiler was called for"""
    (tmp_path / "csrc").mkdir()
    for f in ("one.hip", "two.hip", "head.h"):
        (tmp_path / "csrc" / f).write_text("")
    log = tmp_path / "calls"
    cc = tmp_path / "cc"
    # stands for hipcc: notes its output's name, leaves its arguments there; fails where the file `broken` names the output
    cc.write_text('#!/bin/sh\nfor a; do [ "$p" = "-o" ] && o=$a; p=$a; done\nbasename "$o" >> %s\necho "$@" > "$o"\n'
                  '[ "$(cat %s 2>/dev/null)" != "$(basename "$o")" ]\n' % (log, tmp_path / "broken"))
    cc.chmod(cc.stat().st_mode | stat.S_IEXEC)
    monkeypatch.setenv("HIPCC", str(cc))
    for name, value in (("HERE", str(tmp_path)), ("CSRC", str(tmp_path / "csrc")), ("LIB", str(tmp_path / "lib" / "lib.so")),
                        ("SOURCES", ["one.hip", "two.hip"]), ("HEADERS", ["head.h"])):
        monkeypatch.setattr(b, name, value)

    def run(**kw):
        log.write_text("")
        b.build(**kw)
        return sorted(log.read_text().split())

    run.path = tmp_path
    return run


def test_nothing_is_compiled_twice(tree):
    assert tree() == ["lib.so", "one.o", "two.o"]
    assert tree() == []
    assert tree(force=True) == ["lib.so", "one.o", "two.o"]


def test_a_newer_source_or_header_is_compiled_again(tree):
    tree()
    later = os.path.getmtime(tree.path / "lib" / "lib.so") + 10
    os.utime(tree.path / "csrc" / "one.hip", (later, later))
    assert tree() == ["lib.so", "one.o"]
    os.utime(tree.path / "csrc" / "head.h", (later, later))
    assert tree() == ["lib.so", "one.o", "two.o"]


def test_other_flags_compile_everything_again(tree, monkeypatch):
    tree()
    monkeypatch.setattr(b, "FLAGS", b.FLAGS + ["-DOTHER"])
    assert tree() == ["lib.so", "one.o", "two.o"]
    assert "-DOTHER" in (tree.path / "lib" / "obj" / "two.o").read_text()
    assert tree() == []


def test_a_changed_list_of_sources_links_again(tree, monkeypatch):
    tree()
    monkeypatch.setattr(b, "SOURCES", ["one.hip"])
    assert tree() == ["lib.so"]


def test_an_object_of_a_failed_run_is_compiled_again(tree):
    (tree.path / "broken").write_text("two.o\n")
    with pytest.raises(RuntimeError):
        tree()
    (tree.path / "broken").unlink()
    assert tree() == ["lib.so", "two.o"]   # (the failed run left a two.o that is newer than its source)


def test_the_build_check_compiles_every_time(monkeypatch):
    """__graft_entry__.build() answers "does it build": built files that are there do not answer it"""
    import __graft_entry__ as g
    seen = []
    monkeypatch.setattr(b, "build", lambda force=False, verbose=False: seen.append(force) or b.LIB)
    g.build()
    assert seen == [True]
