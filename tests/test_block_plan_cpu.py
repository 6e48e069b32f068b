"""CPU test of the choice among the forms of a product of blocks of 128 (the library's own code, compiled for the host): the forms that the GPU
tests name run under the shapes that they use, K is cut in 2, 4 and 8 parts among them, and what only pairs of CTAs can take goes there."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
SMS = 148


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "block_plan_selftest"
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-o", str(exe), os.path.join(ROOT, "tests", "host", "block_plan_selftest.cpp")])

    def call(m, n, k, experts=0, pairs_only=False, block_rows=0, split_k=0, cta_pair=0):
        line = f"{m} {max(experts, 1)} {n} {k} {int(experts > 0)} {int(pairs_only)} {block_rows} {split_k} {cta_pair} {SMS}\n"
        return tuple(int(v) for v in subprocess.run([str(exe)], input=line, check=True, capture_output=True, text=True).stdout.split())

    return call


def test_named_forms_are_those_that_run(plan):
    for m, n, k in ((16, 272, 7168), (16, 4096, 7168), (64, 144, 8192), (300, 272, 7680), (129, 400, 2304), (40, 272, 8192)):
        for rows in (16, 32, 64):
            assert plan(m, n, k, block_rows=rows, split_k=1) == (rows, 1)
        assert plan(m, n, k, cta_pair=1) == (0, 1)
    for m, n, k in ((16, 272, 7168), (16, 4096, 7168), (64, 144, 8192), (129, 400, 2304), (40, 272, 8192)):
        assert plan(m, n, k, block_rows=16, split_k=8) == (16, 8)
        assert plan(m, n, k, block_rows=32, split_k=2) == (32, 2)
        assert plan(m, n, k, block_rows=64, split_k=4) == (64, 4)
    assert plan(400, 272, 7168, experts=4, block_rows=32, split_k=2) == (32, 2)
    assert plan(400, 272, 7168, experts=4, block_rows=64, split_k=4) == (64, 4)


def test_parts_have_a_block_and_room(plan):
    assert plan(16, 128, 128, block_rows=16, split_k=8) == (16, 1)
    assert plan(16, 128, 129 * 16, block_rows=16) == (16, 8)
    assert plan(16, 128, 300 // 16 * 16, block_rows=16) == (16, 2)  # three blocks
    for m in (1, 16, 100, 1000):
        for n in (16, 1024, 4096, 16384):
            rows, parts = plan(m, n, 7168, block_rows=64)
            tiles = -(-m // 64) * -(-n // 128)
            assert rows == 64 and parts in (1, 2, 4, 8) and (parts == 1 or tiles * parts <= 2 * SMS)


def test_only_pairs_take_columns(plan):
    for m in (16, 144, 4096):
        for options in (dict(block_rows=16), dict(block_rows=64, split_k=4), dict(cta_pair=2), dict()):
            assert plan(m, 272, 8192, pairs_only=True, **options) == (0, 1)


def test_automatic_choices(plan):
    assert plan(16, 4096, 7168) == (16, 8)  # a decode step
    assert plan(8192, 2304, 7168) == (0, 1) and plan(3001, 7168, 2304) == (0, 1)
    assert plan(128, 4096, 7168, experts=32)[0] in (16, 32) and plan(16384, 2304, 7168, experts=32) == (0, 1)
    assert plan(2**31 - 256, 16, 16)[1] == 1 and plan(2**31 - 256, 16, 16, experts=1024)[1] == 1
