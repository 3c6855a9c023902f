"""Building the library and the extension of the block operators' calls: several
processes of a job may find them stale at the same time."""
import os
import subprocess
import types

import pytest

from qwen_imager_b200 import build


@pytest.fixture
def out(tmp_path, monkeypatch):
    """Builds go to an empty folder."""
    monkeypatch.setattr(build, "OUT_DIR", str(tmp_path))
    monkeypatch.setattr(build, "HOST", str(tmp_path / "_qmm_host.so"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "libqmm.so"))
    return tmp_path


@pytest.mark.parametrize("what", ["build_host", "build"])
def test_builds_at_the_same_time_do_not_share_files(out, monkeypatch, what):
    target = build.HOST if what == "build_host" else build.LIB
    written, nested = [], []

    def compiler(cmd, **kw):
        made = cmd[cmd.index("-o") + 1]
        assert os.path.abspath(made) != target          # published whole, by a rename
        written.append(made)
        open(made, "w").write("half")
        if not nested:                                  # another process builds from start to end meanwhile
            nested.append(True)
            getattr(build, what)(force=True)
            assert open(target).read() == "whole"
            assert open(made).read() == "half"          # and leaves this one's files alone
        open(made, "w").write("whole")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    monkeypatch.setattr(build, "sources", lambda: ["one.cu"])
    assert getattr(build, what)(force=True) == target
    assert open(target).read() == "whole"
    assert len(set(written)) == len(written)
    assert os.listdir(out) == [os.path.basename(target)]


@pytest.mark.parametrize("what", ["build_host", "build"])
def test_a_failed_build_leaves_what_was_there(out, monkeypatch, what):
    target = build.HOST if what == "build_host" else build.LIB
    open(target, "w").write("before")

    def compiler(cmd, **kw):
        open(cmd[cmd.index("-o") + 1], "w").write("half")
        return subprocess.CompletedProcess(cmd, 1, "", "")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    monkeypatch.setattr(build, "sources", lambda: ["one.cu"])
    with pytest.raises(RuntimeError):
        getattr(build, what)(force=True)
    assert open(target).read() == "before" and os.listdir(out) == [os.path.basename(target)]
