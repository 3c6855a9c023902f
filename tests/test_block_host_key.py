"""The extension of the block operators' calls is loaded only as built from the present
sources and for the present torch: it fills the argument structs of the headers that
it was compiled against, so another one would pass misplaced pointers."""
import os
import shutil

import pytest
import torch

from qwen_imager_b200 import _block, build


def test_the_built_extension_holds_the_present_key():
    assert _block.host().key == build.host_key()
    assert not build.host_is_stale()


@pytest.mark.parametrize("change", ["source", "header", "torch"])
def test_another_source_or_torch_makes_it_stale(change, tmp_path, monkeypatch):
    _block.host()
    newer = str(tmp_path / "_qmm_host.so")
    shutil.copy(build.HOST, newer)                       # younger than every source
    monkeypatch.setattr(build, "HOST", newer)
    assert not build.host_is_stale()
    if change == "torch":
        monkeypatch.setattr(torch, "__version__", "0.0")
    elif change == "source":
        other = tmp_path / "block_host.cpp"
        other.write_text(open(build.HOST_SRC).read() + "\n")
        os.utime(other, (0, 0))
        monkeypatch.setattr(build, "HOST_SRC", str(other))
    else:
        include = tmp_path / "include"
        shutil.copytree(os.path.join(build.ROOT, "include"), include)
        with open(include / "qmm_block.h", "a") as f:
            f.write("\n")
        os.utime(include / "qmm_block.h", (0, 0))
        monkeypatch.setattr(build, "ROOT", str(tmp_path))
    assert build.host_is_stale()


def test_a_stale_one_that_cannot_be_rebuilt_is_not_loaded(tmp_path, monkeypatch):
    _block.host()
    stale = str(tmp_path / "_qmm_host.so")
    shutil.copy(build.HOST, stale)
    monkeypatch.setattr(build, "HOST", stale)
    monkeypatch.setattr(build, "host_key", lambda: "another")

    def failing(force=False):
        raise RuntimeError("no compiler")

    monkeypatch.setattr(build, "build_host", failing)
    monkeypatch.setattr(_block, "_host_module", None)
    with pytest.warns(RuntimeWarning, match="no compiler"):
        assert _block.host() is _block._General
