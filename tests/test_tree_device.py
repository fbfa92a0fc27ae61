"""The tree calls launch on their tensors' device, whichever is current: their Python
side over a stand-in for the library, without a GPU."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RUN = """
import ctypes, sys
import torch
lib = ctypes.PyDLL(sys.argv[1])
a, b = (ctypes.c_int * 5)(), (ctypes.c_int * 5)()
lib.tree_devices(a, b)
print(list(a), list(b), flush=True)
"""


def test_calls_launch_on_their_tensors_device(tmp_path):
    pytest.importorskip("torch")
    from tensormark_amd import build

    out = str(tmp_path / "check.so")
    cmd = build.ops_command(out, os.path.join(ROOT, "tests", "cpp", "tree_device_check.cpp"), optimize="-O0", library=False)
    subprocess.run(cmd, check=True)
    got = subprocess.run([sys.executable, "-c", RUN, out], check=True, capture_output=True, text=True, cwd=ROOT).stdout
    assert got.split("\n")[0] == "[1, 1, 1, 1, 1] [0, 0, 0, 0, 0]"
