"""The paged operators without a GPU: the integer code that device kernels
bound their accesses with, the checks of the C ABI and of the Python calls, and
the kernels' resources."""
import ctypes
import json
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from rdnattention import _build

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_rows_stay_in_bounds(tmp_path):
    exe = tmp_path / "paged_rows_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=signed-integer-overflow",
                    "-fno-sanitize-recover=all", f"-I{ROOT / 'rdnattention_amd' / 'csrc'}",
                    str(ROOT / "tests" / "cxx" / "paged_rows_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok ") and int(r.stdout.split()[1]) > 100000


# ---------------------------------------------------------------------------
# C ABI: refused before any HIP call
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    if not _build.LIB.exists():
        _build.build()
    from rdnattention import paged

    return paged._handle()


_hold = ctypes.create_string_buffer(4096 + 64)
_P = (ctypes.addressof(_hold) + 63) // 64 * 64


class _Cache(ctypes.Structure):
    """rdna_paged_cache (include/rdnattention_ext.h)."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("key", "value", "key_scale", "value_scale", "block_tables", "seq_lens",
                                                "cu_seqlens")] +
                [(f"{n}_stride_{a}", ctypes.c_int64) for n in ("key", "value", "key_scale", "value_scale")
                 for a in ("page", "token", "head")] +
                [("table_stride", ctypes.c_int64)] +
                [(n, ctypes.c_uint32) for n in ("num_pages", "page_size", "table_width", "num_seqs", "num_kv_heads",
                                                "head_dim")] +
                [("dtype", ctypes.c_int32)])


def test_packed_cache_has_the_layout_of_the_struct():
    from rdnattention.paged import _CACHE

    values = list(range(1, 28))
    names = [n for n, _ in _Cache._fields_]
    assert len(names) == len(values)
    c = _Cache.from_buffer_copy(_CACHE.pack(*values).ljust(ctypes.sizeof(_Cache), b"\0"))
    assert [getattr(c, n) for n in names] == values


def cache(**kw):
    c = _Cache(key=_P, value=_P, block_tables=_P, seq_lens=_P, num_pages=4, page_size=16, table_width=3, num_seqs=2,
               num_kv_heads=2, head_dim=64, dtype=0, table_stride=3)
    for n in ("key", "value"):
        for a, x in (("page", 2048), ("token", 128), ("head", 64)):
            setattr(c, f"{n}_stride_{a}", x)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def attention(lib, c, **kw):
    a = dict(query=_P, output=_P, qs=256, qh=64, os=256, oh=64, rows=4, heads=4, dtype=0, most=4, scale=0.1, causal=1,
             window=-1, tree=None, tsb=0, tsr=0, tn=0, zero=0)
    a.update(kw)
    rc = lib.rdna_paged_attention(ctypes.addressof(c) if c is not None else None, *a.values(), None)
    return rc, lib.rdna_get_error().decode()


def append(lib, c, **kw):
    a = dict(key=_P, value=_P, ks=128, kh=64, vs=128, vh=64, rows=4, dtype=0, query=None, out=None, qs=256, qh=64,
             os=256, oh=64, heads=4, pos=None, cos=None, sin=None, rot_rows=8, rot_dim=64, pairs=1)
    a.update(kw)
    rc = lib.rdna_paged_append(ctypes.addressof(c) if c is not None else None, *a.values(), None)
    return rc, lib.rdna_get_error().decode()


def commit(lib, c, **kw):
    a = dict(prefix=_P, path=_P, stride=4, n=4, lens=_P)
    a.update(kw)
    rc = lib.rdna_paged_commit(ctypes.addressof(c) if c is not None else None, *a.values(), None)
    return rc, lib.rdna_get_error().decode()


BAD_CACHES = [
    (dict(dtype=3), "cache dtype"), (dict(head_dim=48), "head_dim"), (dict(head_dim=288), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(dtype=2, head_dim=96), "int8"), (dict(num_kv_heads=0), "num_kv_heads"),
    (dict(num_seqs=0), "empty launch grid"), (dict(num_seqs=2 ** 24 + 1), "num_seqs"), (dict(page_size=0), "page_size"),
    (dict(page_size=24), "page_size"), (dict(page_size=2 ** 21), "page_size"),
    (dict(table_width=2 ** 25), "2^28 keys"), (dict(num_pages=0), "num_pages"), (dict(num_pages=2 ** 31), "num_pages"),
    (dict(key=None), "null cache"), (dict(value=None), "null cache"), (dict(block_tables=None), "null cache"),
    (dict(key=_P + 8), "16-byte"), (dict(value=_P + 2), "16-byte"), (dict(block_tables=_P + 2), "block_tables"),
    (dict(table_stride=-1), "block_tables"), (dict(key_stride_page=2044), "strides"),
    (dict(value_stride_token=-128), "strides"), (dict(key_stride_head=4), "strides"),
    (dict(value_stride_head=2 ** 41), "strides"), (dict(dtype=2), "key_scale and value_scale"),
    (dict(dtype=2, key_scale=_P, value_scale=_P + 2), "aligned float"),
    (dict(dtype=2, key_scale=_P, value_scale=_P, key_scale_stride_page=-1), "scale strides"),
]


@pytest.mark.parametrize("kw,message", BAD_CACHES)
def test_abi_refuses_caches(lib, kw, message):
    for call, name in ((attention, "attention"), (append, "append"), (commit, "commit")):
        rc, err = call(lib, cache(**kw))
        assert rc == -3 and err.startswith(f"Paged {name} failed: ") and message in err, err


def test_abi_refuses_a_null_cache(lib):
    for call in (attention, append, commit):
        rc, err = call(lib, None)
        assert rc == -3 and "null cache" in err


@pytest.mark.parametrize("kw,message", [
    (dict(dtype=2), "fp16 or bf16"), (dict(dtype=1), "type of the pages"), (dict(rows=0), "empty launch grid"),
    (dict(rows=2 ** 28 + 2), "2^28"), (dict(rows=5), "multiple of num_seqs")])
def test_abi_refuses_rows(lib, kw, message):
    for call in (attention, append):
        rc, err = call(lib, cache(), **kw)
        assert rc == -3 and message in err, err
    for call in (attention, append):
        rc, err = call(lib, cache(seq_lens=None))
        assert rc == -3 and "null seq_lens" in err


@pytest.mark.parametrize("kw,message", [
    (dict(heads=0), "num_heads"), (dict(heads=3), "num_heads"), (dict(heads=65536), "num_heads"),
    (dict(rows=2 ** 28, heads=16), "2^30"), (dict(query=None), "null tensor"), (dict(output=None), "null tensor"),
    (dict(query=_P + 8), "16-byte"), (dict(output=_P + 8), "16-byte"), (dict(qs=4), "strides"),
    (dict(oh=-64), "strides"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"),
    (dict(tree=_P, tn=4), "tree mask"), (dict(tree=_P, tn=4, causal=0, window=3), "tree mask"),
    (dict(tree=_P, tn=0, causal=0), "tree_n"), (dict(tree=_P, tn=4, tsb=-1, causal=0), "tree_n")])
def test_abi_refuses_attention(lib, kw, message):
    rc, err = attention(lib, cache(), **kw)
    assert rc == -3 and message in err, err


@pytest.mark.parametrize("kw,message", [
    (dict(key=None), "null tensor"), (dict(value=None), "null tensor"), (dict(key=_P + 2), "16-byte"),
    (dict(ks=4), "strides"), (dict(vh=-64), "strides"), (dict(cos=_P), "both"), (dict(query=_P), "rot_cos"),
    (dict(pos=_P), "rot_cos"), (dict(cos=_P, sin=_P + 4), "16-byte"), (dict(cos=_P, sin=_P, rot_dim=8), "rot_dim"),
    (dict(cos=_P, sin=_P, rot_dim=80), "rot_dim"), (dict(cos=_P, sin=_P, rot_dim=0), "rot_dim"),
    (dict(cos=_P, sin=_P, rot_rows=0), "rot_rows"), (dict(cos=_P, sin=_P, query=_P), "query_out"),
    (dict(cos=_P, sin=_P, query=_P, out=_P, heads=0), "num_heads"),
    (dict(cos=_P, sin=_P, query=_P, out=_P, qs=4), "strides"), (dict(rows=2 ** 28), "2^34")])
def test_abi_refuses_appends(lib, kw, message):
    rc, err = append(lib, cache(), **kw)
    assert rc == -3 and message in err, err


@pytest.mark.parametrize("kw,message", [
    (dict(prefix=None), "null index"), (dict(path=None), "null index"), (dict(lens=None), "null index"),
    (dict(path=_P + 2), "aligned"), (dict(n=0), "path_n"), (dict(n=1025), "path_n"), (dict(stride=-1), "path_stride")])
def test_abi_refuses_commits(lib, kw, message):
    rc, err = commit(lib, cache(), **kw)
    assert rc == -3 and message in err, err
    rc, err = commit(lib, cache(num_seqs=65536))
    assert rc == -3 and "65535" in err


# ---------------------------------------------------------------------------
# Python calls
# ---------------------------------------------------------------------------
def tensors(**kw):
    t = dict(key_cache=torch.zeros(4, 16, 2, 64, dtype=torch.float16),
             value_cache=torch.zeros(4, 16, 2, 64, dtype=torch.float16),
             block_tables=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32))
    t.update(kw)
    return t


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


BAD_TENSORS = [
    (dict(key_cache=None), TypeError, "key_cache"), (dict(value_cache=3), TypeError, "value_cache"),
    (dict(key_cache=torch.zeros(4, 16, 64).half()), ValueError, "4D"),
    (dict(key_cache=torch.zeros(4, 16, 64, 2).half().transpose(2, 3)), ValueError, "contiguous head_dim"),
    (dict(value_cache=torch.zeros(4, 16, 1, 64).half()), ValueError, "value_cache must have the shape"),
    (dict(value_cache=torch.zeros(4, 16, 2, 64).bfloat16()), ValueError, "value_cache must have the shape"),
    (dict(key_cache=torch.zeros(4, 16, 2, 64), value_cache=torch.zeros(4, 16, 2, 64)), ValueError, "float16, bfloat16"),
    (dict(key_cache=torch.zeros(4, 16, 2, 64).char(), value_cache=torch.zeros(4, 16, 2, 64).char()), ValueError,
     "key_scale and value_scale"),
    (dict(key_scale=torch.zeros(4, 16, 2)), ValueError, "int8 pages"),
    (dict(key_cache=torch.zeros(4, 16, 2, 64).char(), value_cache=torch.zeros(4, 16, 2, 64).char(),
          key_scale=torch.zeros(4, 16, 2), value_scale=torch.zeros(4, 16, 3)), ValueError, "value_scale"),
    (dict(key_cache=torch.zeros(4, 12, 2, 64).half(), value_cache=torch.zeros(4, 12, 2, 64).half()), ValueError,
     "power of two"),
    (dict(key_cache=torch.zeros(0, 16, 2, 64).half(), value_cache=torch.zeros(0, 16, 2, 64).half()), ValueError,
     "pages and heads"),
    (dict(block_tables=torch.zeros(2, 3, dtype=torch.int64)), ValueError, "int32"),
    (dict(block_tables=i32(6)), ValueError, "2D"), (dict(block_tables=i32(3, 2).t()), ValueError, "contiguous rows"),
    (dict(seq_lens=i32(3)), ValueError, "seq_lens"), (dict(seq_lens=i32(4)[::2]), ValueError, "contiguous"),
    (dict(seq_lens=torch.zeros(2)), ValueError, "int32"),
]


@pytest.mark.parametrize("kw,exc,message", BAD_TENSORS)
def test_python_refuses_caches(kw, exc, message):
    import rdnattention as ra

    t = tensors(**kw)
    rows = torch.zeros(4, 2, 64, dtype=torch.float16)
    for call in (lambda: ra.paged_attention(rows, **t), lambda: ra.paged_append(rows, rows, **t),
                 lambda: ra.paged_tree_attention(rows, tree_mask=torch.ones(2, 2, 2, dtype=torch.bool), **t)):
        with pytest.raises(exc, match=message):
            call()
    lens = t.pop("seq_lens")
    if message in ("seq_lens", "int32", "contiguous"):
        message = "prefix_lens|seq_lens|int32|contiguous"
    with pytest.raises(exc, match=message):
        ra.paged_commit(prefix_lens=lens, path=i32(2, 4), path_lens=i32(2), **t)


def test_python_refuses_unsupported_head_dims():
    import rdnattention as ra

    rows = torch.zeros(4, 2, 48, dtype=torch.float16)
    bad = torch.zeros(4, 16, 2, 48, dtype=torch.float16)
    with pytest.raises(ra.RDNAttentionError, match="head_dim 48"):
        ra.paged_attention(rows, **tensors(key_cache=bad, value_cache=bad))
    bad = torch.zeros(4, 16, 2, 96, dtype=torch.int8)
    sc = torch.zeros(4, 16, 2)
    with pytest.raises(ra.RDNAttentionError, match="int8"):
        ra.paged_attention(rows, **tensors(key_cache=bad, value_cache=bad, key_scale=sc, value_scale=sc))


def test_python_refuses_cpu_tensors():
    """Valid but for the device: the last check."""
    import rdnattention as ra

    rows = torch.zeros(4, 2, 64, dtype=torch.float16)
    for call in (lambda: ra.paged_attention(rows, **tensors()), lambda: ra.paged_append(rows, rows, **tensors())):
        with pytest.raises(ValueError, match="HIP device"):
            call()


@pytest.mark.parametrize("kw,message", [
    (dict(cu_seqlens_q=i32(2)), "cu_seqlens_q must have 3"), (dict(cu_seqlens_q=i32(1, 3)), "1D"),
    (dict(query=torch.zeros(4, 128).half()), "3D"), (dict(query=torch.zeros(5, 2, 64).half()), "divide"),
    (dict(query=torch.zeros(4, 3, 64).half()), "multiple of kv heads"),
    (dict(query=torch.zeros(4, 2, 32).half()), "shape"), (dict(query=torch.zeros(4, 2, 64).bfloat16()), "float16"),
    (dict(query=torch.zeros(4, 64, 2).half().transpose(1, 2)), "contiguous head_dim"),
    (dict(out=torch.zeros(4, 1, 64).half()), "out must"), (dict(out=torch.zeros(4, 2, 64)), "out must")])
def test_python_refuses_rows(kw, message):
    import rdnattention as ra

    t = tensors(query=torch.zeros(4, 2, 64, dtype=torch.float16))
    t.update(kw)
    with pytest.raises(ValueError, match=message):
        ra.paged_attention(**t)


def mask(*shape):
    return torch.ones(*shape, dtype=torch.bool)


@pytest.mark.parametrize("tree,exc,message", [
    (None, TypeError, "tree_mask"), (torch.ones(2, 2, 2), ValueError, "bool"), (mask(2, 2), ValueError, "3D"),
    (mask(1, 2, 2), ValueError, "shape"), (mask(2, 2, 3), ValueError, "shape"), (mask(2, 1, 1), ValueError, "covers"),
    (mask(2, 3, 3).transpose(1, 2), ValueError, "contiguous rows")])
def test_python_refuses_trees(tree, exc, message):
    import rdnattention as ra

    with pytest.raises(exc, match=message):
        ra.paged_tree_attention(torch.zeros(4, 2, 64).half(), tree_mask=tree, **tensors())


@pytest.mark.parametrize("kw,message", [
    (dict(value=torch.zeros(3, 2, 64).half()), "value must have shape"),
    (dict(value=torch.zeros(4, 2, 64).bfloat16()), "value must be"),
    (dict(rot_cos=torch.zeros(9, 32)), "both"), (dict(query=torch.zeros(4, 4, 64).half()), "need rot_cos"),
    (dict(positions=i32(4)), "need rot_cos"),
    (dict(rot_cos=torch.zeros(9, 32), rot_sin=torch.zeros(8, 32)), "same shape"),
    (dict(rot_cos=torch.zeros(9, 32).half(), rot_sin=torch.zeros(9, 32)), "float32"),
    (dict(rot_cos=torch.zeros(9, 4), rot_sin=torch.zeros(9, 4)), "rot_dim"),
    (dict(rot_cos=torch.zeros(9, 40), rot_sin=torch.zeros(9, 40)), "rot_dim"),
    (dict(rot_cos=torch.zeros(0, 32), rot_sin=torch.zeros(0, 32)), "rot_dim"),
    (dict(rot_cos=torch.zeros(9, 32), rot_sin=torch.zeros(9, 32), positions=i32(3)), "positions"),
    (dict(rot_cos=torch.zeros(9, 32), rot_sin=torch.zeros(9, 32), query=torch.zeros(3, 4, 64).half()), "query")])
def test_python_refuses_appends(kw, message):
    import rdnattention as ra

    rows = torch.zeros(4, 2, 64, dtype=torch.float16)
    a = dict(key=rows, value=rows, **tensors())
    a.update(kw)
    with pytest.raises(ValueError, match=message):
        ra.paged_append(**a)


@pytest.mark.parametrize("kw,message", [
    (dict(path=i32(3, 4)), "one row per sequence"), (dict(path_lens=i32(3)), "one row per sequence"),
    (dict(path=i32(2, 1025)), "1024"), (dict(path=i32(4, 2).t()), "contiguous rows"),
    (dict(path=torch.zeros(2, 4)), "int32")])
def test_python_refuses_commits(kw, message):
    import rdnattention as ra

    t = tensors()
    a = dict(key_cache=t["key_cache"], value_cache=t["value_cache"], block_tables=t["block_tables"],
             prefix_lens=t["seq_lens"], path=i32(2, 4), path_lens=i32(2))
    a.update(kw)
    with pytest.raises(ValueError, match=message):
        ra.paged_commit(**a)


def test_kernels_do_not_spill():
    """The kernels of every head dim and type, and the waves that one of their
    workgroups puts on a SIMD."""
    if not _build.RESOURCES.exists():
        _build.build()
    ks = [k for k in json.loads(_build.RESOURCES.read_text()) if "paged_" in k["kernel"]]
    for t in ("DF16_", "DF16b"):
        for d in range(32, 257, 32):
            for base in ("12paged_stream", "11paged_tiles"):
                assert any(f"{base}I{t}Li{d}ELb0E" in k["kernel"] for k in ks), (base, t, d)
        for d in (64, 128):
            for base in ("12paged_stream", "11paged_tiles"):
                assert any(f"{base}I{t}Li{d}ELb1E" in k["kernel"] for k in ks), (base, t, d)
    for k in ks:
        assert k.get("scratch_bytes_per_lane", 0) == 0 and k["lds_bytes"] <= 160 * 1024, k
