"""The index arithmetic of paged attention's workgroups (csrc/attention_place.h) compiled for the host: no starts, in
whatever order, lead to rows outside the call."""

import shutil
import subprocess
from pathlib import Path

import pytest

TESTS = Path(__file__).resolve().parent
CSRC = TESTS.parent / "m5-max-kernels_amd" / "csrc"


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_rows_stay_inside_the_call(tmp_path):
    program = tmp_path / "check"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{CSRC}",
                    str(TESTS / "attention_place_check.cpp"), "-o", str(program)], check=True)
    run = subprocess.run([str(program)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout + run.stderr
