"""The exchange between a pair's two softmax groups (csrc/softmax_pair.cuh), run on the host.

A group that decides to rescale passes one barrier more than one that does not. The two groups therefore have to decide
alike in every order that the barriers themselves allow, with anything in the place where the other pair leaves its
references: that is what they meet once a bounded wait of the kernel has run out.
"""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def test_both_groups_of_a_pair_decide_alike_in_any_order(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = tmp_path / "softmax_pair_check"
    subprocess.run([cxx, "-O1", "-std=c++17", "-Wall", "-I", str(ROOT / "halo_flash_b200" / "csrc"), "-o", str(exe),
                    str(ROOT / "tests" / "cpu" / "softmax_pair_check.cpp")], check=True)
    tiles, bad = map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    assert tiles == 40000 and bad == 0
