"""Blocks of keys and entries of prefixes as the paged kernels deal them, on the host, and the
refusal of key weights whose blocks 32 bits do not count."""
import shutil
import subprocess
from pathlib import Path

import pytest

from tests.test_paged_evict_host import weights
from tests.test_paged_host import cache, lib  # noqa: F401

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_items(tmp_path):
    exe = tmp_path / "paged_items_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=signed-integer-overflow",
                    "-fno-sanitize-recover=all", f"-I{ROOT / 'rdnattention_amd' / 'csrc'}",
                    str(ROOT / "tests" / "cxx" / "paged_items_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok ") and int(r.stdout.split()[1]) > 1000000


def test_abi_refuses_too_many_blocks(lib):  # noqa: F811
    """One sequence of 2^24 rows of two heads over a table of 2^26 keys: 2^20 row tiles for each
    of 2^19 blocks, by the kernel of many rows alone."""
    rc, err = weights(lib, cache(num_seqs=1, table_width=2 ** 22), rows=2 ** 24)
    assert rc == -3 and "key tiles" in err, err
