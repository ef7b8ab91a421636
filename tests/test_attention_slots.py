"""The slots that paged attention's workgroups are numbered by (csrc/attention_place.h), on the host: enough for every
tile, and none without rows for a call of single tokens."""

import shutil
import subprocess
from pathlib import Path

import pytest

TESTS = Path(__file__).resolve().parent
CSRC = TESTS.parent / "m5-max-kernels_amd" / "csrc"


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_slots_hold_every_tile(tmp_path):
    program = tmp_path / "check"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{CSRC}",
                    str(TESTS / "attention_slots_check.cpp"), "-o", str(program)], check=True)
    run = subprocess.run([str(program)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout + run.stderr
