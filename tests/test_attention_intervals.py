"""Which keys a row of dense attention sees and which rows see a key, against the definition (attention_intervals_check.cpp), on the CPU."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_rows_and_keys_see_each_other(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    exe = str(tmp_path / "check")
    # (an overflow of 32 bits ends the program)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all", "-o", exe, os.path.join(HERE, "attention_intervals_check.cpp")], check=True, timeout=120)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr
