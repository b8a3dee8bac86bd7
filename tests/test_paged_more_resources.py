"""Registers and LDS of the paged kernels for norms, prefixes, weights of keys and eviction: the
waves that a CU is meant to hold (CPU only: the compiler's remarks of the last build)."""
import json
import re

import pytest

from rdnattention import _build

LDS = 160 * 1024


@pytest.fixture(scope="module")
def kernels():
    if not _build.RESOURCES.exists():
        _build.build()
    return json.loads(_build.RESOURCES.read_text())


def _of(kernels, pattern):
    found = [(m, k) for k in kernels if (m := re.search(r"\d+" + pattern, k["kernel"]))]
    return found


def test_joins(kernels):
    """Eight waves of a workgroup, two to a SIMD, up to head_dim 128, four above that."""
    found = _of(kernels, r"(paged_join_stream|paged_join_tiles)IDF16b?_?Li(\d+)ELb([01])E(?:Li([48])E)?")
    for m, k in found:
        d = int(m.group(2))
        assert k["waves_per_simd"] >= (2 if d <= 128 else 1) and k["lds_bytes"] <= LDS, k
        assert m.group(4) in (None, "8" if d <= 128 else "4"), k["kernel"]
    assert len(found) == 2 * 2 * 10  # 8 head dims and 2 of int8 pages, of two types


def test_rows_with_a_log_sum_exp(kernels):
    """As many waves as the calls without (paged_stream)."""
    found = _of(kernels, r"paged_out_stream(IDF16b?_?Li(\d+)ELb[01]ELi([48])E)")
    for m, k in found:
        (_, plain), = _of(kernels, "paged_stream" + m.group(1))
        assert k["waves_per_simd"] == plain["waves_per_simd"], (k, plain)
    assert len(found) == 2 * (10 + 3)


def test_weights(kernels):
    """Few rows: eight waves of one workgroup up to head_dim 128, four above; many: two workgroups
    of four waves, or one."""
    found = _of(kernels, r"paged_weights_(few|many)IDF16b?_?Li(\d+)ELb([01])E")
    for m, k in found:
        narrow = int(m.group(2)) <= 128
        assert k["waves_per_simd"] >= (2 if narrow else 1), k
        assert k["lds_bytes"] * (2 if narrow and m.group(1) == "many" else 1) <= LDS, k
    assert len(found) == 2 * 2 * 10


def test_norms(kernels):
    """Five waves of 16-bit rows on a SIMD, two where keys are quantised (in fp64)."""
    found = _of(kernels, r"paged_append_normedIDF16b?_?Lb([01])ELi(\d+)ELi(\d+)E")
    for m, k in found:
        assert k["waves_per_simd"] >= (2 if m.group(1) == "1" else 5), k
    assert len(found) == 2 * 2 * (4 + 2)


def test_eviction(kernels):
    """Workgroups of 1024 threads: of short tables two on a CU, else one; two of moves."""
    for pattern, groups in ((r"paged_evict_chooseILi8192E", 2), (r"paged_evict_chooseILi34816E", 1),
                            (r"paged_evict_moveE", 2)):
        (_, k), = _of(kernels, pattern)
        assert k["waves_per_simd"] >= 4 * groups and k["lds_bytes"] * groups <= LDS, k
