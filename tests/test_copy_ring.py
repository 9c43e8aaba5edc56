"""The count of copies through a ring (csrc/exl3cu_ring.h), compiled for the host: which barrier phase each wait is for, and
that the copy whose wait gave up is waited for once more with those behind it."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    exe = tmp_path_factory.mktemp("ring") / "copy_ring_check"
    subprocess.run([gxx, "-std=c++17", "-Wall", "-Werror", f"-I{ROOT / 'xiaomi-hexagon-exl3_b200' / 'csrc'}",
                    str(ROOT / "tests" / "cpp" / "copy_ring_check.cpp"), "-o", str(exe)], check=True)
    return lambda *a: subprocess.run([str(exe), *map(str, a)], check=True, capture_output=True, text=True).stdout.strip()


def phase(i, stages):
    return f"{i % stages}{i // stages & 1}"


@pytest.mark.parametrize("stages", [2, 3])
@pytest.mark.parametrize("copies", [0, 1, 2, 3, 7, 8])
def test_every_copy_is_waited_for_in_its_phase(check, stages, copies):
    got, drained = check(stages, copies, -1).split("|") if copies else ("", check(stages, 0, -1).strip("| "))
    assert got.split() == [phase(i, stages) for i in range(copies)] and not drained.split()


@pytest.mark.parametrize("stages", [2, 3])
@pytest.mark.parametrize("copies,fails", [(1, 0), (2, 0), (2, 1), (8, 0), (8, 3), (8, 7), (3, 2)])
def test_what_did_not_arrive_is_drained(check, stages, copies, fails):
    got, drained = (x.split() for x in check(stages, copies, fails).split("|"))
    assert got == [phase(i, stages) for i in range(fails + 1)]
    assert drained == [phase(i, stages) for i in range(fails, min(copies, fails + stages))]
