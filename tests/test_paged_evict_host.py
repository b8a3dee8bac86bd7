"""The refusals of paged_key_weights and paged_evict, and which rows see a key, without a
GPU."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from tests.test_paged_host import BAD_CACHES, _P, cache, i32, lib, tensors  # noqa: F401

ROOT = Path(__file__).resolve().parent.parent
STRIDE = (ctypes.c_int64 * 3)(32, 2, 1)
S = ctypes.addressof(STRIDE)
BAD = (ctypes.c_int64 * 3)(32, -2, 1)


def weights(lib, c, **kw):  # noqa: F811
    a = dict(query=_P, qs=256, qh=64, rows=4, heads=4, dtype=0, most=4, lse=_P, scale=0.1, causal=1, window=-1,
             decay=1.0, w=_P, stride=S)
    a.update(kw)
    rc = lib.rdna_paged_key_weights(ctypes.addressof(c) if c is not None else None, *a.values(), None)
    return rc, lib.rdna_get_error().decode()


def evict(lib, c, **kw):  # noqa: F811
    a = dict(w=_P, stride=S, budget=8, first=1, recent=2, lens=_P + 512, kept=_P)
    a.update(kw)
    rc = lib.rdna_paged_evict(ctypes.addressof(c) if c is not None else None, *a.values(), None)
    return rc, lib.rdna_get_error().decode()


@pytest.mark.parametrize("kw,message", [x for x in BAD_CACHES if "value" not in str(x[0])])
def test_abi_refuses_caches(lib, kw, message):  # noqa: F811
    for call, name in ((weights, "key weights"), (evict, "evict")):
        rc, err = call(lib, cache(**kw))
        assert rc == -3 and err.startswith(f"Paged {name} failed: ") and message in err, err
        rc, err = call(lib, None)
        assert rc == -3 and "null cache" in err


@pytest.mark.parametrize("kw,message", [
    (dict(heads=0), "num_heads"), (dict(heads=3), "num_heads"), (dict(heads=65536), "num_heads"),
    (dict(rows=2 ** 28, heads=16), "2^30"), (dict(query=None), "null tensor"), (dict(lse=None), "null tensor"),
    (dict(query=_P + 8), "16-byte"), (dict(lse=_P + 2), "4-byte"), (dict(qs=4), "strides"), (dict(qh=-64), "strides"),
    (dict(scale=float("nan")), "scale"), (dict(decay=-0.5), "decay"), (dict(decay=float("inf")), "decay"),
    (dict(decay=float("nan")), "decay"), (dict(w=None), "null key_weights"), (dict(stride=None), "null key_weights"),
    (dict(w=_P + 2), "aligned float"), (dict(stride=ctypes.addressof(BAD)), "strides of key_weights"),
    (dict(dtype=2), "fp16 or bf16"), (dict(dtype=1), "type of the pages"), (dict(rows=0), "empty launch grid"),
    (dict(rows=5), "multiple of num_seqs")])
def test_abi_refuses_weights(lib, kw, message):  # noqa: F811
    rc, err = weights(lib, cache(), **kw)
    assert rc == -3 and message in err, err


def test_abi_refuses_too_many_tiles(lib):  # noqa: F811
    # 2^16 sequences, 2 heads, tables of 2^26 keys
    rc, err = weights(lib, cache(num_seqs=2 ** 16, table_width=2 ** 22), rows=2 ** 16)
    assert rc == -3 and "key tiles" in err, err


@pytest.mark.parametrize("kw,message", [
    (dict(w=None), "null key_weights"), (dict(w=_P + 1), "aligned float"),
    (dict(stride=ctypes.addressof(BAD)), "strides of key_weights"), (dict(budget=0), "budget must be"),
    (dict(budget=2 ** 28 + 1), "budget must be"), (dict(first=7), "exceed budget"), (dict(recent=2 ** 32 - 1), "exceed budget"),
    (dict(lens=None), "null index"), (dict(kept=None), "null index"), (dict(lens=_P + 2), "aligned"),
    (dict(kept=_P + 2), "aligned"), (dict(lens=_P), "must not be seq_lens")])
def test_abi_refuses_evictions(lib, kw, message):  # noqa: F811
    rc, err = evict(lib, cache(value=_P + 1024), **kw)
    assert rc == -3 and message in err, err


def test_abi_refuses_more_evictions(lib):  # noqa: F811
    rc, err = evict(lib, cache(num_seqs=65536))
    assert rc == -3 and "65535" in err
    rc, err = evict(lib, cache(seq_lens=None))
    assert rc == -3 and "null index" in err
    rc, err = evict(lib, cache())
    assert rc == -3 and "same memory" in err


W = torch.zeros(4, 16, 2)


@pytest.mark.parametrize("kw,exc,message", [
    (dict(query=3), TypeError, "query"), (dict(lse=None), TypeError, "lse"), (dict(lse=torch.zeros(4, 3)), ValueError, "lse"),
    (dict(lse=torch.zeros(4, 4).half()), ValueError, "lse"), (dict(lse=torch.zeros(4, 8)[:, ::2]), ValueError, "contiguous"),
    (dict(query=torch.zeros(4, 3, 64).half(), lse=torch.zeros(4, 3)), ValueError, "multiple of kv heads"),
    (dict(query=torch.zeros(5, 4, 64).half()), ValueError, "divide among"), (dict(key_weights=None), TypeError, "key_weights"),
    (dict(key_weights=W[:, :, :1]), ValueError, "key_weights"), (dict(key_weights=W.half()), ValueError, "key_weights"),
    (dict(decay=-1.0), ValueError, "decay"), (dict(decay=float("nan")), ValueError, "decay"),
    (dict(key_scale=W), ValueError, "int8 pages"), (dict(seq_lens=i32(3)), ValueError, "seq_lens"),
    (dict(key_cache=None), TypeError, "key_cache")])
def test_python_refuses_weights(kw, exc, message):
    import rdnattention as ra

    a = dict(tensors(), query=torch.zeros(4, 4, 64).half(), lse=torch.zeros(4, 4), key_weights=W)
    a.pop("value_cache")
    a.update(kw)
    with pytest.raises(exc, match=message):
        ra.paged_key_weights(**a)


@pytest.mark.parametrize("kw,exc,message", [
    (dict(budget=0), ValueError, "budget must be"), (dict(budget=-3), ValueError, "budget must be"),
    (dict(budget=2 ** 28 + 1), ValueError, "budget must be"), (dict(first=-1), ValueError, "first"),
    (dict(recent=-1), ValueError, "recent"), (dict(first=5, recent=4), ValueError, "exceed budget"),
    (dict(key_weights=W.double()), ValueError, "key_weights"), (dict(key_weights=7), TypeError, "key_weights"),
    (dict(value_cache=None), TypeError, "value_cache"), (dict(block_tables=i32(6)), ValueError, "2D")])
def test_python_refuses_evictions(kw, exc, message):
    import rdnattention as ra

    a = dict(tensors(), key_weights=W, budget=8)
    a.update(kw)
    with pytest.raises(exc, match=message):
        ra.paged_evict(**a)


def test_nothing_to_do():
    import rdnattention as ra

    t = tensors()
    t.pop("value_cache")
    assert ra.paged_key_weights(torch.zeros(0, 4, 64).half(), torch.zeros(0, 4), key_weights=W, **t) is None
    lens, kept = ra.paged_evict(**tensors(block_tables=i32(0, 3), seq_lens=i32(0)), key_weights=W, budget=8)
    assert lens.shape == (0,) and kept.shape == (0, 2, 8)


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_rows_that_see_a_key(tmp_path):
    exe = tmp_path / "paged_key_rows_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=signed-integer-overflow",
                    "-fno-sanitize-recover=all", f"-I{ROOT / 'rdnattention_amd' / 'csrc'}",
                    str(ROOT / "tests" / "cxx" / "paged_key_rows_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok ")


def test_refuses_expanded_weights(lib):  # noqa: F811
    import rdnattention as ra

    for i in range(3):  # one memory for several weights
        stride = (ctypes.c_int64 * 3)(*(0 if j == i else s for j, s in enumerate((32, 2, 1))))
        for call in (weights, evict):
            rc, err = call(lib, cache(value=_P + 1024), stride=ctypes.addressof(stride))
            assert rc == -3 and "memory of its own" in err, err
        shape = [1 if j == i else n for j, n in enumerate(W.shape)]
        w = torch.zeros(shape).expand(W.shape)
        with pytest.raises(ValueError, match="expanded"):
            ra.paged_evict(**tensors(), key_weights=w, budget=8)
        with pytest.raises(ValueError, match="expanded"):
            a = dict(tensors(), query=torch.zeros(4, 4, 64).half(), lse=torch.zeros(4, 4), key_weights=w)
            a.pop("value_cache")
            ra.paged_key_weights(**a)


def test_refuses_a_decay_beyond_float():
    import rdnattention as ra

    a = dict(tensors(), query=torch.zeros(4, 4, 64).half(), lse=torch.zeros(4, 4), key_weights=W)
    a.pop("value_cache")
    with pytest.raises(ValueError, match="decay"):
        ra.paged_key_weights(**a, decay=1e300)
