"""The check of arguments for shared memory (csrc/overlap.h) against sets of bytes, on the host."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def test_views_overlap_where_their_bytes_do(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = tmp_path / "overlap_check"
    subprocess.run([cxx, "-O2", "-std=c++17", "-Wall", "-I", str(ROOT / "halo_flash_b200" / "csrc"), "-o", str(exe),
                    str(ROOT / "tests" / "cpu" / "overlap_check.cpp")], check=True)
    pairs, bad, bad_self, meet = map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    assert pairs == 30000 and bad == 0 and bad_self == 0 and 5000 < meet < 25000
