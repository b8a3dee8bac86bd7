"""The refusals of paged_append's norms and axes, without a GPU."""
import ctypes

import pytest
import torch

from tests.test_paged_host import _P, cache, i32, lib, tensors  # noqa: F401


class _Norm(ctypes.Structure):
    """rdna_paged_norm (include/rdnattention_ext.h)."""

    _fields_ = [("query_norm", ctypes.c_void_p), ("key_norm", ctypes.c_void_p), ("rot_axes", ctypes.c_void_p),
                ("position_stride", ctypes.c_int64), ("num_axes", ctypes.c_uint32), ("eps", ctypes.c_float),
                ("dtype", ctypes.c_int32)]


def test_packed_norm_has_the_layout_of_the_struct():
    from rdnattention.paged import _NORM

    n = _Norm.from_buffer_copy(_NORM.pack(1, 2, 3, 4, 5, 0.5, 7).ljust(ctypes.sizeof(_Norm), b"\0"))
    assert [getattr(n, f) for f, _ in _Norm._fields_] == [1, 2, 3, 4, 5, 0.5, 7]


ROPE = dict(cos=_P, sin=_P)
QUERY = dict(query=_P, out=_P)


@pytest.mark.parametrize("norm,kw,message", [
    (dict(query_norm=_P), {}, "query_norm without query"),
    (dict(key_norm=_P, dtype=1), {}, "norm weights must be fp32 or"),
    (dict(key_norm=_P, dtype=2), {}, "norm weights must be fp32 or"),
    (dict(key_norm=_P + 4), {}, "norm weights must be 16-byte"),
    (dict(query_norm=_P + 8), QUERY, "norm weights must be 16-byte"),
    (dict(key_norm=_P, eps=-1.0), {}, "eps"), (dict(key_norm=_P, eps=float("nan")), {}, "eps"),
    (dict(key_norm=_P, eps=float("inf")), {}, "eps"),
    (dict(rot_axes=_P, num_axes=3), ROPE, "rot_axes needs"),
    (dict(rot_axes=_P, num_axes=3), dict(pos=_P), "rot_cos"),
    (dict(rot_axes=_P + 2, num_axes=3), dict(ROPE, pos=_P), "aligned int32"),
    (dict(rot_axes=_P, num_axes=0), dict(ROPE, pos=_P), "num_axes"),
    (dict(rot_axes=_P, num_axes=2 ** 16 + 1), dict(ROPE, pos=_P), "num_axes"),
    (dict(rot_axes=_P, num_axes=3, position_stride=-3), dict(ROPE, pos=_P), "position_stride"),
    (dict(rot_axes=_P, num_axes=3, position_stride=2 ** 41), dict(ROPE, pos=_P), "position_stride"),
    (dict(key_norm=_P), QUERY, "rot_cos"), (dict(), dict(key=None), "null tensor"),
    (dict(), dict(rows=5), "multiple of num_seqs"), (dict(key_norm=_P), dict(rows=2 ** 28), "2^34"),
])
def test_abi_refuses(lib, norm, kw, message):  # noqa: F811
    n = _Norm(dtype=3, eps=1e-6, position_stride=3)
    for k, v in norm.items():
        setattr(n, k, v)
    a = dict(key=_P, value=_P, ks=128, kh=64, vs=128, vh=64, rows=4, dtype=0, query=None, out=None, qs=256, qh=64,
             os=256, oh=64, heads=4, pos=None, cos=None, sin=None, rot_rows=8, rot_dim=64, pairs=1)
    a.update(kw)
    c = cache(value=_P + 1024)
    rc = lib.rdna_paged_append_norm(ctypes.addressof(c), ctypes.addressof(n), *a.values(), None)
    err = lib.rdna_get_error().decode()
    assert rc == -3 and err.startswith("Paged append failed: ") and message in err, err


def test_abi_refuses_values_in_the_place_of_keys(lib):  # noqa: F811
    n = _Norm(dtype=3, eps=1e-6)
    c = cache(value=_P)
    assert c.key == c.value
    rc = lib.rdna_paged_append_norm(ctypes.addressof(c), ctypes.addressof(n), _P, _P, 128, 64, 128, 64, 4, 0, None, None,
                                    256, 64, 256, 64, 4, None, None, None, 8, 64, 1, None)
    assert rc == -3 and "same memory" in lib.rdna_get_error().decode()


H = torch.float16


@pytest.mark.parametrize("kw,exc,message", [
    (dict(key_norm=3), TypeError, "key_norm must be a torch.Tensor"),
    (dict(key_norm=torch.ones(63)), ValueError, "key_norm must be"),
    (dict(key_norm=torch.ones(1, 64)), ValueError, "key_norm must be"),
    (dict(key_norm=torch.ones(64, dtype=torch.bfloat16)), ValueError, "key_norm must be"),
    (dict(key_norm=torch.ones(64, dtype=torch.float64)), ValueError, "key_norm must be"),
    (dict(key_norm=torch.ones(128)[::2]), ValueError, "key_norm must be contiguous"),
    (dict(query_norm=torch.ones(64)), ValueError, "query_norm needs query"),
    (dict(query_norm=torch.ones(64), key_norm=torch.ones(64, dtype=H), query=torch.zeros(4, 4, 64, dtype=H)),
     ValueError, "same dtype"),
    (dict(key_norm=torch.ones(64), norm_eps=-1.0), ValueError, "norm_eps"),
    (dict(key_norm=torch.ones(64), norm_eps=float("nan")), ValueError, "norm_eps"),
    (dict(key_norm=torch.ones(64), query=torch.zeros(4, 4, 64, dtype=H)), ValueError, "need rot_cos"),
    (dict(rot_axes=i32(32)), ValueError, "rot_axes needs"),
    (dict(rot_axes=i32(32), positions=i32(4, 3)), ValueError, "need rot_cos"),
    (dict(rot_axes=i32(32), positions=i32(4), rope=1), ValueError, "2D"),
    (dict(rot_axes=i32(31), positions=i32(4, 3), rope=1), ValueError, "rot_axes must have"),
    (dict(rot_axes=i32(32).long(), positions=i32(4, 3), rope=1), ValueError, "rot_axes must be int32"),
    (dict(rot_axes=i32(32), positions=i32(5, 3), rope=1), ValueError, "one entry per row"),
    (dict(rot_axes=i32(32), positions=i32(3, 4).t(), rope=1), ValueError, "contiguous rows"),
    (dict(rot_axes=i32(32), positions=i32(4, 0), rope=1), ValueError, "axes"),
    (dict(positions=i32(4, 3), rope=1), ValueError, "1D"),
    (dict(rot_axes=i32(32), rope=1), ValueError, "rot_axes needs"),
])
def test_python_refuses(kw, exc, message):
    import rdnattention as ra

    rows = torch.zeros(4, 2, 64, dtype=H)
    if kw.pop("rope", 0):
        kw = dict(kw, rot_cos=torch.zeros(8, 32), rot_sin=torch.zeros(8, 32))
    with pytest.raises(exc, match=message):
        ra.paged_append(rows, rows, **tensors(), **kw)


def test_nothing_to_do():
    """No rows, no sequences."""
    import rdnattention as ra

    w = torch.ones(64)
    none = torch.zeros(0, 2, 64, dtype=H)
    assert ra.paged_append(none, none, **tensors(), query=torch.zeros(0, 4, 64, dtype=H), query_norm=w).shape == (0, 4, 64)
    q = torch.randn(4, 4, 64).half()
    t = tensors(block_tables=i32(0, 3), seq_lens=i32(0))
    rows = torch.zeros(4, 2, 64, dtype=H)
    got = ra.paged_append(rows, rows, **t, query=q, query_norm=w, key_norm=w, cu_seqlens_q=i32(1))
    assert torch.equal(got, q)


def test_refuses_an_eps_beyond_float():
    import rdnattention as ra

    rows = torch.zeros(4, 2, 64, dtype=H)
    with pytest.raises(ValueError, match="norm_eps"):
        ra.paged_append(rows, rows, **tensors(), key_norm=torch.ones(64), norm_eps=1e300)
