"""The arithmetic with which launches find their work, compiled from the kernels' own header and
compared with plain division and counting on the host."""

import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "sglang-mlx_amd", "csrc")


def check(tmp_path, header_dir):
    exe = str(tmp_path / "check")
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", str(header_dir), os.path.join(HERE, "schedule_check.cpp"), "-o", exe],
                   check=True)
    return subprocess.run([exe], capture_output=True, text=True)


def test_schedule(tmp_path):
    r = check(tmp_path, CSRC)
    assert r.returncode == 0 and r.stdout == "as counted\n", r.stdout


@pytest.mark.parametrize("right,wrong", [
    ("((uint64_t)1 << (31 + r.shift)) + (uint64_t)d - 1) / (uint64_t)d", "((uint64_t)1 << (31 + r.shift))) / (uint64_t)d"),
    ("(((int64_t)1 << 32) + units - 1) / units", "((int64_t)1 << 32) / units"),
    ("(end - snap) / span", "end / span"),
    ("kScaledStart + snap + span - 1", "snap + span - 1"),
])
def test_the_check_finds_mistakes(tmp_path, right, wrong):
    """Planted in a copy of the header."""
    with open(os.path.join(CSRC, "pkv_schedule.h")) as f:
        text = f.read()
    assert text.count(right) == 1
    (tmp_path / "pkv_schedule.h").write_text(text.replace(right, wrong))
    shutil.copy(os.path.join(HERE, "schedule_check.cpp"), tmp_path)
    r = check(tmp_path, tmp_path)
    assert r.returncode == 1 and r.stdout != "as counted\n"
