"""CPU test of the table of tensor maps: its host code, compiled for a stand-in of the map."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_threads_get_their_own_maps(tmp_path):
    exe = tmp_path / "map_cache_selftest"
    src = os.path.join(ROOT, "tests", "host", "map_cache_selftest.cpp")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-pthread", "-o", str(exe), src])
    assert "map cache ok" in subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=120).stdout
