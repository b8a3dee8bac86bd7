"""Limits of the paged operators' C ABI, refused before any HIP call (CPU)."""
import pytest

from tests.test_paged_host import _P, append, attention, cache, commit, lib  # noqa: F401

FAR = 2 ** 39  # elements


@pytest.mark.parametrize("kw,message", [
    (dict(num_pages=2 ** 31 - 1, key_stride_page=FAR), "strides"),
    (dict(num_pages=2 ** 31 - 1, value_stride_page=2 ** 25), "strides"),
    (dict(page_size=2 ** 20, value_stride_token=2 ** 36), "strides"),
    (dict(num_kv_heads=65535, key_stride_head=2 * FAR), "strides"),  # 65535 * 2^41 bytes
    (dict(num_seqs=2 ** 16, table_stride=2 ** 39), "block_tables"),
    (dict(num_seqs=2 ** 16, table_stride=2 ** 38 + 1), "block_tables"),
    (dict(dtype=2, key_scale=_P, value_scale=_P, num_pages=2 ** 31 - 1, key_scale_stride_page=2 ** 24), "scale strides"),
    (dict(dtype=2, key_scale=_P, value_scale=_P, num_pages=2 ** 31 - 1, value_scale_stride_page=FAR),
     "scale strides")])
def test_no_offset_in_the_cache_leaves_63_bits(lib, kw, message):  # noqa: F811
    """An index times its stride, in bytes, reaches 2^56 at most."""
    rows = kw.get("num_seqs", 2)
    for call in (attention, append, commit):
        more = dict(heads=kw.get("num_kv_heads", 2), rows=rows) if call is attention else \
            dict(rows=rows) if call is append else {}
        if call is commit and kw.get("num_seqs", 0) > 65535:
            kw = dict(kw, num_seqs=65535, table_stride=2 ** 39)
        rc, err = call(lib, cache(**kw), **more)
        assert rc == -3 and message in err and "2^56" in err, err


@pytest.mark.parametrize("kw", [dict(qs=2 ** 31), dict(os=2 ** 31), dict(qh=2 ** 40, heads=65534),
                                dict(tree=_P, tn=2 ** 20, tsr=2 ** 40, causal=0),
                                dict(tree=_P, tn=4, tsb=2 ** 41, causal=0)])
def test_no_offset_in_the_rows_leaves_63_bits(lib, kw):  # noqa: F811
    if "heads" not in kw and "tree" not in kw:
        kw = dict(kw, rows=2 ** 28, heads=2)
    rc, err = attention(lib, cache(), **kw)
    assert rc == -3 and "strides" in err and "2^56" in err, err
    if "qs" in kw:
        rc, err = append(lib, cache(), rows=2 ** 20, ks=2 ** 36)
        assert rc == -3 and "strides" in err and "2^56" in err, err
        rc, err = append(lib, cache(), rows=2 ** 20, cos=_P, sin=_P, query=_P, out=_P, os=2 ** 36)
        assert rc == -3 and "strides" in err and "2^56" in err, err


def test_no_offset_in_the_paths_leaves_63_bits(lib):  # noqa: F811
    rc, err = commit(lib, cache(num_seqs=65535), stride=2 ** 39)
    assert rc == -3 and "path_stride" in err and "2^56" in err, err


@pytest.mark.parametrize("kw", [dict(os=320), dict(oh=128), dict(qs=512, qh=128)])
def test_queries_in_place_need_their_own_strides(lib, kw):  # noqa: F811
    """Rows that lie elsewhere in the same memory would be written over before
    they are read."""
    rc, err = append(lib, cache(), cos=_P, sin=_P, query=_P, out=_P, **kw)
    assert rc == -3 and "query's strides" in err, err


@pytest.mark.parametrize("seqs,rows,heads,width,page", [
    (65536, 65600, 32, 128, 1024),  # too many for the kernel of few rows only, which is launched second
    (1, 2 ** 20, 64, 64, 2 ** 20), (2 ** 24, 2 ** 24 + 1, 32, 2 ** 10, 2 ** 18)])
def test_calls_too_large_are_refused_whole(lib, seqs, rows, heads, width, page):  # noqa: F811
    """Before the first launch: without a device any HIP call would give another
    error."""
    c = cache(num_seqs=seqs, num_kv_heads=8, table_width=width, page_size=page, cu_seqlens=_P, table_stride=width)
    rc, err = attention(lib, c, rows=rows, heads=heads, most=rows)
    assert rc == -3 and "key tiles" in err, err


def test_keys_and_values_in_one_memory_are_not_written(lib):  # noqa: F811
    """The workgroups that move keys and those that move values do not wait for
    each other: in one memory a commit would read what it has already moved."""
    for call in (append, commit):
        rc, err = call(lib, cache())
        assert rc == -3 and "same memory" in err, err
