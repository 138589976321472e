"""What a build reuses and what it compiles again, with a compiler that only notes its calls."""

import os
import stat

import pytest

from vilbert_multi_task_amd.ops import build as ops_build

COMPILER = """#!/bin/sh
echo "$@" >> {log}
if [ -e {fail} ]; then exit 1; fi
while [ $# -gt 0 ]; do
  if [ "$1" = -o ]; then echo built > "$2"; fi
  shift
done
"""


@pytest.fixture
def box(tmp_path, monkeypatch):
    csrc, out = tmp_path / "csrc", tmp_path / "out"
    csrc.mkdir()
    for name in ("a.hip", "b.hip", "c.cpp", "h.h"):
        (csrc / name).write_text(name)
    log, fail, hipcc = tmp_path / "log", tmp_path / "fail", tmp_path / "hipcc"
    hipcc.write_text(COMPILER.format(log=log, fail=fail))
    hipcc.chmod(hipcc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("HIPCC", str(hipcc))
    for name, value in (
        ("CSRC", str(csrc)), ("OUT_DIR", str(out)), ("OBJ_DIR", str(out / "obj")),
        ("OUT_SO", str(out / "lib.so")), ("SOURCES", ["a.hip", "b.hip", "c.cpp"]), ("HEADERS", ["h.h"]),
    ):
        monkeypatch.setattr(ops_build, name, value)
    old = 1_000_000_000
    for path in csrc.iterdir():
        os.utime(path, (old, old))

    class Box:
        so = out / "lib.so"

        def run(self, **kwargs):
            """The commands of a build: of compiling, and of linking."""
            log.write_text("")
            ops_build.build(verbose=False, **kwargs)
            lines = log.read_text().splitlines()
            return [c for c in lines if " -c " in c], [c for c in lines if " -c " not in c]

        def touch(self, name):
            later = self.so.stat().st_mtime + 100
            os.utime(csrc / name, (later, later))

        def break_compiler(self, broken):
            fail.write_text("") if broken else fail.unlink()

        def lose(self, name):
            (csrc / name).unlink()

    return Box()


def test_a_second_build_does_nothing(box):
    compiled, linked = box.run()
    assert len(compiled) == 3 and len(linked) == 1
    assert box.run() == ([], [])
    assert not ops_build.needs_build()
    compiled, linked = box.run(force=True)
    assert len(compiled) == 3 and len(linked) == 1


def test_an_edited_source_is_compiled_alone_and_a_header_for_all(box):
    box.run()
    box.touch("b.hip")
    assert ops_build.needs_build()
    compiled, linked = box.run()
    assert len(compiled) == 1 and "b.hip" in compiled[0] and len(linked) == 1
    box.touch("h.h")
    assert len(box.run()[0]) == 3


@pytest.mark.parametrize("kind", ["asan", "ubsan"])
def test_instrumented_objects_are_not_linked_into_a_plain_build(box, kind):
    compiled, linked = box.run(force=True, **{kind: True})
    assert len(compiled) == 3 and all("-fsanitize=" in c for c in compiled + linked)
    assert ops_build.needs_build()
    compiled, linked = box.run()
    assert len(compiled) == 3 and len(linked) == 1
    assert not any("-fsanitize=" in c for c in compiled + linked)
    compiled, linked = box.run(**{kind: True})  # and back, without force
    assert len(linked) == 1 and "-fsanitize=" in linked[0]


def test_another_architecture_or_compiler_builds_anew(box, monkeypatch, tmp_path):
    box.run()
    monkeypatch.setattr(ops_build, "ARCH", "gfx950:sramecc+")
    assert ops_build.needs_build()
    compiled, linked = box.run()
    assert len(compiled) == 3 and len(linked) == 1
    other = tmp_path / "other"
    other.write_text((tmp_path / "hipcc").read_text())
    other.chmod(0o755)
    monkeypatch.setenv("HIPCC", str(other))
    assert len(box.run()[0]) == 3


def test_objects_of_unknown_make_are_compiled_again(box):
    """What lies there from before says nothing of how it was compiled."""
    os.makedirs(ops_build.OBJ_DIR)
    for name in ops_build.SOURCES:
        with open(os.path.join(ops_build.OBJ_DIR, name + ".o"), "w") as f:
            f.write("old")
    box.so.write_text("old")
    assert ops_build.needs_build()
    assert len(box.run()[0]) == 3


def test_a_failed_build_leaves_the_library_and_is_repeated(box):
    box.run()
    box.so.write_text("the one that works")
    box.touch("a.hip")
    box.break_compiler(True)
    with pytest.raises(Exception):
        box.run()
    assert box.so.read_text() == "the one that works"
    box.break_compiler(False)
    compiled, linked = box.run()
    assert len(compiled) == 1 and len(linked) == 1


def test_a_missing_source_is_an_error(box):
    box.run()
    box.lose("c.cpp")
    with pytest.raises(FileNotFoundError):
        box.run()


@pytest.mark.parametrize("jobs", ["0", "1", "", "64"])
def test_any_number_of_jobs(box, monkeypatch, jobs):
    monkeypatch.setenv("MAX_JOBS", jobs)
    assert len(box.run()[0]) == 3
