"""The build where torch or g++ is not there: the library, which needs neither, without the
Python side of the cache calls."""
from __future__ import annotations

import os
import shutil
import sys

import pytest

from tensormark_amd import build


@pytest.fixture
def small(tmp_path, monkeypatch):
    """A build of one source into a folder of its own."""
    monkeypatch.setattr(build, "BUILD_DIR", str(tmp_path / "objects"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "libtmsample_hip.so"))
    monkeypatch.setattr(build, "OPS", str(tmp_path / "_cache_ops.so"))
    monkeypatch.setattr(build, "SOURCES", ["tms_history.cpp"])
    return tmp_path


@pytest.mark.parametrize("missing", ["torch", "g++"])
def test_the_library_builds_without(small, monkeypatch, capsys, missing):
    (small / "_cache_ops.so").write_bytes(b"of another build")
    if missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    else:
        monkeypatch.setattr(shutil, "which", lambda name: None)
    assert build.build() == str(small / "libtmsample_hip.so")
    assert os.path.exists(build.LIB) and not os.path.exists(build.OPS)
    assert missing in capsys.readouterr().err
