"""Whether two strided operands share memory, on the CPU (plast_amd/csrc/places.hpp, built with g++ into a small program that
counts bytes)."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_places(tmp_path):
    exe = tmp_path / "places_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", f"-I{ROOT / 'include'}",
                    f"-I{ROOT / 'plast_amd' / 'csrc'}", str(ROOT / "tests" / "places_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
