"""Registers of the paged attention kernels: the waves that a CU is meant to hold
(CPU only: the compiler's remarks of the last build)."""
import json
import re

import pytest

from rdnattention import _build


@pytest.fixture(scope="module")
def kernels():
    if not _build.RESOURCES.exists():
        _build.build()
    return json.loads(_build.RESOURCES.read_text())


def test_waves_of_a_simd(kernels):
    """paged_tiles: a workgroup's eight waves are two to a SIMD, above head_dim 128 its
    four one to a SIMD; paged_stream: up to head_dim 128 eight waves on a CU, as one
    workgroup or two, above that four."""
    checked = 0
    for k in kernels:
        m = re.search(r"\d+(paged_stream|paged_tiles)IDF16b?_?Li(\d+)ELb([01])E(?:Li([48])E)?", k["kernel"])
        if m is None:
            continue
        need = 2 if int(m.group(2)) <= 128 else 1
        assert k["waves_per_simd"] >= need, (k["kernel"], k["waves_per_simd"])
        if m.group(1) == "paged_stream" and m.group(4) == "4" and need == 2:
            assert 2 * k["lds_bytes"] <= 160 * 1024, (k["kernel"], k["lds_bytes"])
        checked += 1
    # 8 head dims and 2 of int8 pages of two types; stream at 96, 128 and int8 128 also with eight waves
    assert checked == 2 * (10 + 10 + 3)
