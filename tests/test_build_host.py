"""CPU: what the build compiles again (with a compiler that only writes its output file)."""
import os
import subprocess

import pytest

from vegs_amd import build


@pytest.fixture
def compiled(tmp_path, monkeypatch):
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build.subprocess, "run", run)

    def again(**kw):
        calls.clear()
        build.build(harness=False, **kw)
        return [os.path.basename(c[c.index("-c") + 1]) for c in calls if "-c" in c], len([c for c in calls if "-shared" in c])
    return again


def test_other_flags_compile_everything_again(compiled, monkeypatch):
    everything = (sorted(build.SOURCES), 1)
    first = compiled()
    assert (sorted(first[0]), first[1]) == everything
    assert compiled() == ([], 0)
    monkeypatch.setattr(build, "FLAGS", build.FLAGS + ["-DOTHER"])
    other = compiled()
    assert (sorted(other[0]), other[1]) == everything
    assert compiled() == ([], 0)
    forced = compiled(force=True)
    assert (sorted(forced[0]), forced[1]) == everything


def test_objects_of_unknown_flags_are_compiled_again(compiled):
    compiled()
    os.remove(os.path.join(build.OBJ_DIR, "flags"))
    assert len(compiled()[0]) == len(build.SOURCES)


def test_a_failed_build_is_not_taken_for_a_whole_one(compiled, monkeypatch):
    compiled()
    monkeypatch.setattr(build, "FLAGS", build.FLAGS + ["-DOTHER"])
    works = build.subprocess.run

    def fails(cmd, **kw):
        if "-c" in cmd and cmd[cmd.index("-c") + 1].endswith("xgmi.hip"):
            return subprocess.CompletedProcess(cmd, 1, "", "no")
        return works(cmd, **kw)
    monkeypatch.setattr(build.subprocess, "run", fails)
    with pytest.raises(RuntimeError, match="hipcc failed"):
        compiled()
    monkeypatch.setattr(build.subprocess, "run", works)
    assert len(compiled()[0]) == len(build.SOURCES)
