"""The closing of an aborting SM pair's half-issued stages (csrc/pair_settle.h), on the CPU: a model of the leader's
full barriers under random schedules that stop anywhere (tests/native/pair_settle_check.cpp)."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_stage_ends_with_its_last_copy(tmp_path):
    exe = tmp_path / "pair_settle_check"
    src = os.path.join(HERE, "native", "pair_settle_check.cpp")
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", str(exe), src], check=True)
    r = subprocess.run([str(exe), "200000"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.strip() == "200000 schedules, 0 wrong"
