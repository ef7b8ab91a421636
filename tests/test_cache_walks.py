"""The heads that the workgroups of cache_walk_cases.py's calls walk over (csrc/cache_walk.h), on the host."""

import shutil
import subprocess
from pathlib import Path

import pytest

from cache_walk_cases import CASES, HEADS

TESTS = Path(__file__).resolve().parent
CSRC = TESTS.parent / "m5-max-kernels_amd" / "csrc"


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    program = tmp_path_factory.mktemp("walk") / "check"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{CSRC}", str(TESTS / "cache_walk_check.cpp"),
                    "-o", str(program)], check=True)
    return lambda *a: int(subprocess.run([str(program), *map(str, a)], check=True, capture_output=True, text=True).stdout)


@pytest.mark.parametrize("name", CASES)
def test_cases_walk_over_heads(name, walk):
    c = CASES[name]
    append = walk("append", sum(c["new"]), c["block"], HEADS, c["hq"], c["threads"])
    read = walk("read", sum(c["new"]), c["d"], HEADS)
    assert (append, read) == (c["append"], c["read"])
    assert min(append, read) > 1 and HEADS % append and HEADS % read


def test_small_calls_do_not_walk(walk):
    assert walk("append", 64, 16, 8, 56, 256) == 1 and walk("read", 64, 128, 8) == 1
    assert walk("append", 1 << 28, 16, 64, 64, 1024) == 8 and walk("read", 1 << 28, 128, 64) == 8
