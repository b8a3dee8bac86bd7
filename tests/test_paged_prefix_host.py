"""The refusals of paged_prefix_attention, and which rows a prefix's are, without a GPU."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from tests.test_paged_host import _P, cache, i32, lib, tensors  # noqa: F401

ROOT = Path(__file__).resolve().parent.parent


class _Prefix(ctypes.Structure):
    """rdna_paged_prefix (include/rdnattention_ext.h)."""

    _fields_ = [("block_tables", ctypes.c_void_p), ("lens", ctypes.c_void_p), ("seqs", ctypes.c_void_p),
                ("table_stride", ctypes.c_int64), ("table_width", ctypes.c_uint32), ("num_prefixes", ctypes.c_uint32)]


def test_packed_prefix_has_the_layout_of_the_struct():
    from rdnattention.paged import _PREFIX

    p = _Prefix.from_buffer_copy(_PREFIX.pack(*range(1, 7)).ljust(ctypes.sizeof(_Prefix), b"\0"))
    assert [getattr(p, f) for f, _ in _Prefix._fields_] == [1, 2, 3, 4, 5, 6]


@pytest.mark.parametrize("prefix,kw,message", [
    (dict(num_prefixes=0), {}, "num_prefixes"), (dict(num_prefixes=2 ** 24 + 1), {}, "num_prefixes"),
    (dict(num_prefixes=2, seqs=None), {}, "several prefixes"), (dict(table_width=2 ** 25), {}, "2^28 keys"),
    (dict(lens=None), {}, "null prefix"), (dict(block_tables=None), {}, "null prefix"),
    (dict(lens=_P + 2), {}, "aligned int32"), (dict(seqs=_P + 2), {}, "aligned int32"),
    (dict(block_tables=_P + 1), {}, "aligned int32"), (dict(table_stride=-1), {}, "aligned int32"),
    ({}, dict(window=5), "window_size"), ({}, dict(lse=_P + 2), "lse"), ({}, dict(heads=3), "num_heads"),
    ({}, dict(query=None), "null tensor"), ({}, dict(rows=0), "empty launch grid"),
    # 2^14 prefixes of 2^23 keys each with 4 heads: more key tiles than 32 bits count
    (dict(num_prefixes=2 ** 14, table_width=2 ** 19), dict(rows=2 ** 14), "key tiles"),
])
def test_abi_refuses(lib, prefix, kw, message):  # noqa: F811
    p = _Prefix(block_tables=_P, lens=_P, seqs=_P, table_stride=3, table_width=3, num_prefixes=1)
    for k, v in prefix.items():
        setattr(p, k, v)
    a = dict(query=_P, output=_P, qs=256, qh=64, os=256, oh=64, rows=4, heads=4, dtype=0, most=4, scale=0.1, causal=1,
             window=-1, zero=0, lse=None)
    a.update(kw)
    c = cache()
    rc = lib.rdna_paged_attention_lse(ctypes.addressof(c), ctypes.addressof(p), *a.values(), None)
    err = lib.rdna_get_error().decode()
    assert rc == -3 and err.startswith("Paged attention failed: ") and message in err, err


@pytest.mark.parametrize("kw,exc,message", [
    (dict(prefix_tables=None), TypeError, "prefix_tables"), (dict(prefix_lens=[3]), TypeError, "prefix_lens"),
    (dict(prefix_tables=i32(3)), ValueError, "2D"), (dict(prefix_tables=i32(1, 3).long()), ValueError, "int32"),
    (dict(prefix_lens=i32(2)), ValueError, "prefix_lens must have"),
    (dict(prefix_tables=i32(0, 3), prefix_lens=i32(0)), ValueError, "at least one"),
    (dict(prefix_tables=i32(2, 3), prefix_lens=i32(2)), ValueError, "need prefix_seqs"),
    (dict(prefix_seqs=i32(3)), ValueError, "prefix_seqs must have 2"), (dict(prefix_seqs=[0, 2]), TypeError, "prefix_seqs"),
    (dict(query=torch.zeros(4, 3, 64).half()), ValueError, "multiple of kv heads"),
    (dict(query=torch.zeros(5, 4, 64).half()), ValueError, "divide among"),
    (dict(block_tables=None), TypeError, "block_tables"), (dict(seq_lens=i32(3)), ValueError, "seq_lens"),
])
def test_python_refuses(kw, exc, message):
    import rdnattention as ra

    a = dict(query=torch.zeros(4, 4, 64).half(), prefix_tables=i32(1, 3), prefix_lens=i32(1), **tensors())
    a.update(kw)
    with pytest.raises(exc, match=message):
        ra.paged_prefix_attention(**a)


def test_nothing_to_do():
    import rdnattention as ra

    a = dict(prefix_tables=i32(1, 3), prefix_lens=i32(1), return_lse=True, **tensors())
    out, lse = ra.paged_prefix_attention(torch.zeros(0, 4, 64).half(), **a)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    a.update(block_tables=i32(0, 3), seq_lens=i32(0), cu_seqlens_q=i32(1))
    out, lse = ra.paged_prefix_attention(torch.ones(3, 4, 64).half(), **a)
    assert (out == 0).all() and (lse == float("-inf")).all()


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_rows_of_a_prefix_stay_in_bounds(tmp_path):
    exe = tmp_path / "paged_group_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=signed-integer-overflow",
                    "-fno-sanitize-recover=all", f"-I{ROOT / 'rdnattention_amd' / 'csrc'}",
                    str(ROOT / "tests" / "cxx" / "paged_group_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok ")
