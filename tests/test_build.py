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


def _tool(name):
    import importlib.util
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, "tools", name + ".py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("check", ["hot_loops", "arrival_counter_waits", "mfma_fresh_operand_reads"])
def test_isa_checks_compile_what_is_built(check, monkeypatch):
    """a check of waits and hazards says something of the library only if it compiles the sources with the library's flags"""
    mod, seen = _tool("isa_loop_check"), []

    class Nothing:
        stdout = ""

    monkeypatch.setattr(mod.subprocess, "run", lambda cmd, **kw: seen.append(cmd) or Nothing)
    getattr(mod, check)()
    assert seen and all(all(f in cmd for f in b.FLAGS) for cmd in seen), seen


@pytest.mark.parametrize("script,first", [("build_variant_tu.sh", "act8"), ("build_variant.sh", "pivotcvae_amd/csrc/catalog_bf16.hip")])
def test_variant_libraries_differ_in_one_source_alone(script, first, tmp_path):
    """the variant's own unit with the library's flags (and the given one), and every other object of the library beside it"""
    import subprocess
    log, cc = tmp_path / "calls", tmp_path / "cc"
    cc.write_text('#!/bin/sh\necho "$@" >> %s\n' % log)
    cc.chmod(cc.stat().st_mode | stat.S_IEXEC)
    subprocess.run(["bash", os.path.join(ROOT, "tools", script), first, str(tmp_path / "v.so"), "-DVARIANT"], check=True, cwd=ROOT,
                   env=dict(os.environ, HIPCC=str(cc)), stdout=subprocess.DEVNULL)
    compiled, linked = (line.split() for line in log.read_text().splitlines())
    assert "-DVARIANT" in compiled and all(f in compiled for f in b.FLAGS)
    objects = {os.path.basename(o) for o in linked if o.endswith(".o")}
    own = os.path.splitext(os.path.basename(first))[0] + ".o"
    assert objects == {os.path.splitext(s)[0] + ".o" for s in b.SOURCES} - {own} | {"v.o"}
