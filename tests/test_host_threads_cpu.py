"""CPU tests of what host threads share or have of their own: the tables of tensor maps (host code, compiled for a stand-in of the
map) and the values of a device."""
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


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_values_of_a_device(tmp_path):
    exe = tmp_path / "per_device_selftest"
    src = os.path.join(ROOT, "tests", "host", "per_device_selftest.cpp")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=thread", "-o", str(exe), src])
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    if "FATAL: ThreadSanitizer: unexpected memory mapping" in run.stderr:
        pytest.skip("the race detector cannot run under this kernel's address layout")
    assert run.returncode == 0 and "per device ok" in run.stdout, run.stdout + run.stderr
