"""How the paged attention kernels deal their work, on the host."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_shares(tmp_path):
    exe = tmp_path / "paged_share_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=signed-integer-overflow",
                    "-fno-sanitize-recover=all", f"-I{ROOT / 'rdnattention_amd' / 'csrc'}",
                    str(ROOT / "tests" / "cxx" / "paged_share_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok ") and int(r.stdout.split()[1]) > 100000


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_largest_cost(tmp_path):
    exe = tmp_path / "paged_cost_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=signed-integer-overflow",
                    "-fno-sanitize-recover=all", f"-I{ROOT / 'rdnattention_amd' / 'csrc'}",
                    str(ROOT / "tests" / "cxx" / "paged_cost_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok ") and int(r.stdout.split()[1]) >= 60000
