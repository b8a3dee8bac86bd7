"""Paged key/value caches: appending, attention, trees of drafts, commits.

Keys and values of all sequences live in pages of page_size tokens, a power of
two: ``key_cache`` and ``value_cache`` are [num_pages, page_size, kv_heads,
head_dim] (any strides with a contiguous head_dim axis; transpose a cache kept
as [num_pages, kv_heads, page_size, head_dim]).  ``block_tables`` int32
[sequences, width] lists each sequence's pages in order.  The lengths
``seq_lens`` int32 [sequences] count the keys in the cache, a step's new rows
among them.  Row tensors are [rows, heads, head_dim]: without ``cu_seqlens_q``
every sequence has rows / sequences of them, with it (int32 [sequences + 1])
rows cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1 are sequence b's, and rows
behind the last sequence are padding.  A sequence's n rows are its newest: row
i has index seq_lens[b] - n + i in the sequence.

All of these are tensors on one HIP device; none is read on the host, so calls
neither synchronise nor change under graph capture.  Types: float16 or
bfloat16 rows with pages of the same type, or either with int8 pages and a
float32 scale per token and head (``key_scale``, ``value_scale`` [num_pages,
page_size, kv_heads]; head_dim 64 and 128).  head_dim: multiples of 32 up to
256.  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes

import rdnattention as _ra

SUPPORTED_HEAD_DIMS_PAGED = tuple(range(32, 257, 32))

_VP, _I64, _U32, _I32, _F32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_uint32, ctypes.c_int32, ctypes.c_float


class _Cache(ctypes.Structure):
    """rdna_paged_cache (include/rdnattention_ext.h)."""

    _fields_ = ([(n, _VP) for n in ("key", "value", "key_scale", "value_scale", "block_tables", "seq_lens",
                                    "cu_seqlens")] +
                [(f"{n}_stride_{a}", _I64) for n in ("key", "value", "key_scale", "value_scale")
                 for a in ("page", "token", "head")] +
                [("table_stride", _I64)] +
                [(n, _U32) for n in ("num_pages", "page_size", "table_width", "num_seqs", "num_kv_heads", "head_dim")] +
                [("dtype", _I32)])


_lib = None


def _handle():
    global _lib
    if _lib is None:
        lib = _ra._lib_handle()
        if not hasattr(lib, "rdna_paged_attention"):  # RDNATTENTION_LIB may name an older library
            raise _ra.RDNAttentionError(f"{lib._name} has no paged-cache operators: rebuild it")
        cache = ctypes.POINTER(_Cache)
        lib.rdna_paged_append.argtypes = ([cache, _VP, _VP] + [_I64] * 4 + [_U32, _I32, _VP, _VP] + [_I64] * 4 +
                                          [_U32, _VP, _VP, _VP, _U32, _U32, _I32, _VP])
        lib.rdna_paged_append.restype = _I32
        lib.rdna_paged_attention.argtypes = ([cache, _VP, _VP] + [_I64] * 4 + [_U32, _U32, _I32, _U32, _F32, _I32, _I32,
                                                                              _VP, _I64, _I64, _U32, _I32, _VP])
        lib.rdna_paged_attention.restype = _I32
        lib.rdna_paged_commit.argtypes = [cache, _VP, _VP, _I64, _U32, _VP, _VP]
        lib.rdna_paged_commit.restype = _I32
        _lib = lib
    return _lib


def _index(name, t, dim, device):
    torch = _ra._torch()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} must be {dim}D, got shape {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on the same device as key_cache")
    if dim == 1 and not t.is_contiguous() or dim == 2 and t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have contiguous rows - call .contiguous() first")
    return t.data_ptr()


def _cache(key_cache, value_cache, block_tables, seq_lens, cu_seqlens, key_scale, value_scale, rows):
    """The checked caches and sequences as (_Cache, sequences, kv_heads,
    head_dim)."""
    torch = _ra._torch()
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4D [pages, page_size, kv_heads, head_dim], got shape {tuple(t.shape)}")
        if t.stride(3) != 1:
            raise ValueError(f"{name} must have a contiguous head_dim axis")
    shape = tuple(key_cache.shape)
    dtype = key_cache.dtype
    device = key_cache.device
    if tuple(value_cache.shape) != shape or value_cache.dtype != dtype or value_cache.device != device:
        raise ValueError("value_cache must have the shape, dtype and device of key_cache")
    pages, page_size, kv_heads, head_dim = shape
    if dtype == torch.int8:
        code = 2
        if head_dim not in _ra.SUPPORTED_HEAD_DIMS_INT8:
            raise _ra.RDNAttentionError(f"paged cache: head_dim {head_dim} not supported with int8 pages (64 and 128)")
        if key_scale is None or value_scale is None:
            raise ValueError("int8 pages need key_scale and value_scale")
        for name, t in (("key_scale", key_scale), ("value_scale", value_scale)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if t.dtype != torch.float32 or tuple(t.shape) != shape[:3] or t.device != device:
                raise ValueError(f"{name} must be a float32 tensor of shape {shape[:3]} on the device of key_cache")
        scales = key_scale.data_ptr(), value_scale.data_ptr()
        scale_strides = key_scale.stride() + value_scale.stride()
    else:
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"key_cache must be float16, bfloat16 or int8, got {dtype}")
        if key_scale is not None or value_scale is not None:
            raise ValueError("key_scale and value_scale go with int8 pages")
        if head_dim not in SUPPORTED_HEAD_DIMS_PAGED:
            raise _ra.RDNAttentionError(f"paged cache: head_dim {head_dim} not supported (multiples of 32 from 32 to 256)")
        code = 0 if dtype == torch.float16 else 1
        scales = None, None
        scale_strides = (0,) * 6
    if page_size == 0 or page_size & (page_size - 1) or page_size > 1 << 20:
        raise ValueError(f"page_size must be a power of two up to 2^20, got {page_size}")
    if pages == 0 or kv_heads == 0:
        raise ValueError(f"the caches must have pages and heads, got shape {shape}")
    table = _index("block_tables", block_tables, 2, device)
    seqs, width = tuple(block_tables.shape)
    lens = None
    if seq_lens is not None:
        lens = _index("seq_lens", seq_lens, 1, device)
        if seq_lens.shape[0] != seqs:
            raise ValueError(f"seq_lens must have one entry per row of block_tables ({seqs}), got {seq_lens.shape[0]}")
    cu = None
    if cu_seqlens is not None:
        cu = _index("cu_seqlens_q", cu_seqlens, 1, device)
        if cu_seqlens.shape[0] != seqs + 1:
            raise ValueError(f"cu_seqlens_q must have {seqs + 1} entries, got {cu_seqlens.shape[0]}")
    elif rows is not None and (rows % seqs if seqs else rows):
        raise ValueError(f"{rows} rows do not divide among {seqs} sequences (pass cu_seqlens_q)")
    c = _Cache(key_cache.data_ptr(), value_cache.data_ptr(), *scales, table, lens, cu, *key_cache.stride()[:3],
               *value_cache.stride()[:3], *scale_strides, block_tables.stride(0), pages, page_size, width, seqs, kv_heads,
               head_dim, code)
    return c, seqs, kv_heads, head_dim


def _rows(name, t, shape, cache, like=None):
    """A row tensor: 3D, the given heads and head_dim (None: any), of a type that
    goes with the cache."""
    torch = _ra._torch()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dim() != 3:
        raise ValueError(f"{name} must be 3D [rows, heads, head_dim], got shape {tuple(t.shape)}")
    for have, want in zip(t.shape, shape):
        if want is not None and have != want:
            raise ValueError(f"{name} must have shape {tuple('any' if x is None else x for x in shape)}, "
                             f"got {tuple(t.shape)}")
    if t.dtype not in (torch.float16, torch.bfloat16) or cache.dtype not in (torch.int8, t.dtype):
        raise ValueError(f"{name} must be {'float16 or bfloat16' if cache.dtype == torch.int8 else cache.dtype}, "
                         f"got {t.dtype}")
    if like is not None and t.dtype != like.dtype:
        raise ValueError(f"{name} must be {like.dtype}, got {t.dtype}")
    if t.device != cache.device:
        raise ValueError(f"{name} must be on the same device as key_cache")
    if t.stride(2) != 1:
        raise ValueError(f"{name} must have a contiguous head_dim axis")
    return t.data_ptr()


def _call(device, what, fn, *args):
    """fn(*args, stream) on the device's current stream."""
    torch = _ra._torch()
    if device.type != "cuda":
        raise ValueError(f"{what}: the tensors must be on a HIP device")
    if device.index == torch.cuda.current_device():
        rc = fn(*args, _ra._stream())
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _ra._stream())
    if rc != 0:
        raise _ra.RDNAttentionError(f"{what} failed: {_ra.last_error()}")


def paged_append(key, value, key_cache, value_cache, block_tables, seq_lens, *, cu_seqlens_q=None, query=None,
                 positions=None, rot_cos=None, rot_sin=None, rot_interleaved: bool = True, key_scale=None,
                 value_scale=None):
    """Writes a step's keys and values to their places in the pages, in place.

    key/value: float16 or bfloat16 [rows, kv_heads, head_dim].  int8 pages get
    each row quantised with its own scale, as quantize_int8_qk_pertoken does;
    the scales are written to key_scale and value_scale.

    rot_cos/rot_sin: float32 [positions, rot_dim // 2] RoPE tables (rot_dim a
    multiple of 16 up to head_dim); the first rot_dim channels of the keys are
    rotated on the way, in fp32 and rounded once.  Channels 2i, 2i + 1 turn by
    column i, or with rot_interleaved=False channels i and i + rot_dim // 2.
    The angles are those of the row's index in its sequence, or of positions
    (int32 [rows]: drafts of a tree stand side by side in the cache, not in the
    text); indices outside the tables are taken as their first or last row.

    query: optional [rows, heads, head_dim]; returned rotated likewise, as a new
    tensor.  Padding rows, and rows without a place (a sequence shorter than
    its rows, a page outside the cache), write nothing.  Returns None without
    query."""
    torch = _ra._torch()
    if not isinstance(key, torch.Tensor):
        raise TypeError("key must be a torch.Tensor")
    if key.dim() != 3:
        raise ValueError(f"key must be 3D [rows, heads, head_dim], got shape {tuple(key.shape)}")
    rows = key.shape[0]
    c, _, kv_heads, head_dim = _cache(key_cache, value_cache, block_tables, seq_lens, cu_seqlens_q, key_scale,
                                      value_scale, rows)
    if seq_lens is None:
        raise TypeError("seq_lens must be a torch.Tensor")
    k = _rows("key", key, (rows, kv_heads, head_dim), key_cache)
    v = _rows("value", value, (rows, kv_heads, head_dim), key_cache, key)
    device = key_cache.device
    cos = sin = pos = q = q_out = None
    rot_rows = rot_dim = heads = 0
    q_st = o_st = (0, 0)
    if (rot_cos is None) != (rot_sin is None):
        raise ValueError("pass both rot_cos and rot_sin, or neither")
    if rot_cos is not None:
        for name, t in (("rot_cos", rot_cos), ("rot_sin", rot_sin)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if t.dtype != torch.float32 or t.dim() != 2 or not t.is_contiguous() or t.device != device:
                raise ValueError(f"{name} must be a contiguous 2D float32 tensor on the device of key_cache")
        if rot_cos.shape != rot_sin.shape:
            raise ValueError("rot_cos and rot_sin must have the same shape")
        rot_rows, rot_dim = rot_cos.shape[0], 2 * rot_cos.shape[1]
        if rot_rows == 0 or rot_dim == 0 or rot_dim % 16 or rot_dim > head_dim:
            raise ValueError(f"rot_cos must be [positions, rot_dim // 2], rot_dim a multiple of 16 up to {head_dim}, "
                             f"got {tuple(rot_cos.shape)}")
        cos, sin = rot_cos.data_ptr(), rot_sin.data_ptr()
        if positions is not None:
            pos = _index("positions", positions, 1, device)
            if positions.shape[0] != rows:
                raise ValueError(f"positions must have one entry per row ({rows}), got {positions.shape[0]}")
    elif query is not None or positions is not None:
        raise ValueError("query and positions need rot_cos and rot_sin")
    out = None
    if query is not None:
        q = _rows("query", query, (rows, None, head_dim), key_cache, key)
        heads = query.shape[1]
        out = torch.empty(tuple(query.shape), dtype=query.dtype, device=device)
        if heads == 0:
            q = None
        else:
            q_out, q_st, o_st = out.data_ptr(), query.stride(), out.stride()
    if rows == 0:
        return out
    if c.num_seqs == 0:  # nothing but padding
        return out.copy_(query) if out is not None else None
    ks, vs = key.stride(), value.stride()
    _call(device, "paged_append", _handle().rdna_paged_append, c, k, v, ks[0], ks[1], vs[0], vs[1], rows,
          0 if key.dtype == torch.float16 else 1, q, q_out, q_st[0], q_st[1], o_st[0], o_st[1], heads, pos, cos, sin,
          rot_rows, rot_dim, 1 if rot_interleaved else 0)
    return out


def _attend(what, query, key_cache, value_cache, block_tables, seq_lens, cu_seqlens_q, max_seqlen_q, is_causal,
            window_size, scale, tree_mask, key_scale, value_scale, out):
    torch = _ra._torch()
    if not isinstance(query, torch.Tensor):
        raise TypeError("query must be a torch.Tensor")
    if query.dim() != 3:
        raise ValueError(f"query must be 3D [rows, heads, head_dim], got shape {tuple(query.shape)}")
    rows, heads, _ = query.shape
    c, seqs, kv_heads, head_dim = _cache(key_cache, value_cache, block_tables, seq_lens, cu_seqlens_q, key_scale,
                                         value_scale, rows)
    if seq_lens is None:
        raise TypeError("seq_lens must be a torch.Tensor")
    q = _rows("query", query, (rows, None, head_dim), key_cache)
    if heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a multiple of kv heads ({kv_heads})")
    tree, t_sb, t_sr, t_n = None, 0, 0, 0
    device = key_cache.device
    if tree_mask is not None:
        if not isinstance(tree_mask, torch.Tensor):
            raise TypeError("tree_mask must be a torch.Tensor")
        if tree_mask.dtype != torch.bool or tree_mask.dim() != 3 or tree_mask.device != device:
            raise ValueError("tree_mask must be a 3D bool tensor on the device of key_cache")
        n = tree_mask.shape[1]
        if tree_mask.shape[0] != seqs or tree_mask.shape[2] != n:
            raise ValueError(f"tree_mask must have shape [{seqs}, drafts, drafts], got {tuple(tree_mask.shape)}")
        if cu_seqlens_q is None and seqs and rows // seqs > n:
            raise ValueError(f"tree_mask covers {n} drafts, the call has {rows // seqs} per sequence")
        if n > 1 and tree_mask.stride(2) != 1:
            raise ValueError("tree_mask must have contiguous rows - call .contiguous() first")
        tree, t_sb, t_sr, t_n = tree_mask.data_ptr(), tree_mask.stride(0), tree_mask.stride(1), n
    zero_tail = out is None
    if out is None:
        out = torch.empty(tuple(query.shape), dtype=query.dtype, device=device)
    else:
        _rows("out", out, tuple(query.shape), key_cache, query)
    if out.numel() == 0:
        return out
    if seqs == 0 or t_n == 0 and tree_mask is not None:  # no row is a sequence's, or sees a key
        if tree_mask is not None and seqs:
            raise ValueError("tree_mask covers no draft")
        return out.zero_() if zero_tail else out
    qs, os_ = query.stride(), out.stride()
    most = rows if max_seqlen_q is None else max(0, min(rows, int(max_seqlen_q)))
    _call(device, what, _handle().rdna_paged_attention, c, q, out.data_ptr(), qs[0], qs[1], os_[0], os_[1], rows, heads,
          0 if query.dtype == torch.float16 else 1, most, float(head_dim ** -0.5 if scale is None else scale),
          1 if is_causal else 0, max(-1, min(int(window_size), 2 ** 31 - 1)), tree, t_sb, t_sr, t_n, 1 if zero_tail else 0)
    return out


def paged_attention(query, key_cache, value_cache, block_tables, seq_lens, *, cu_seqlens_q=None, max_seqlen_q=None,
                    is_causal: bool = True, window_size: int = -1, scale=None, key_scale=None, value_scale=None,
                    out=None):
    """Attention of each sequence's newest rows over its pages: single tokens,
    chunks of a prompt, whole prompts, or all of them in one ragged batch.

    query: float16 or bfloat16 [rows, heads, head_dim], a multiple of the
    caches' heads, the rows' keys already appended.  is_causal and window_size
    as in flash_attn, aligned to the end of the keys; a row that sees no key
    comes out as zeros.  scale defaults to 1/sqrt(head_dim).  max_seqlen_q: most
    rows of any sequence (with cu_seqlens_q; default: all rows) - it picks
    kernels and decides no result.

    out: optional tensor like query to write to, whose padding rows stay as they
    are; a new tensor's are zeros.  Returns the output."""
    return _attend("paged_attention", query, key_cache, value_cache, block_tables, seq_lens, cu_seqlens_q, max_seqlen_q,
                   is_causal, window_size, scale, None, key_scale, value_scale, out)


def paged_tree_attention(query, key_cache, value_cache, block_tables, seq_lens, tree_mask, *, cu_seqlens_q=None,
                         max_seqlen_q=None, scale=None, key_scale=None, value_scale=None, out=None):
    """Attention of drafted tokens that form a tree.

    The newest rows of each sequence are its drafts (appended with the
    positions of their depth).  Row i sees every key before the drafts, and
    draft j where tree_mask[b, i, j] (bool [sequences, drafts, drafts]; a draft
    sees itself only if the mask says so).  Sequences with fewer drafts than
    the mask use its first rows and columns; drafts beyond the mask are seen by
    none and see the prefix alone.  The rest as in paged_attention."""
    if tree_mask is None:
        raise TypeError("tree_mask must be a torch.Tensor")
    return _attend("paged_tree_attention", query, key_cache, value_cache, block_tables, seq_lens, cu_seqlens_q,
                   max_seqlen_q, False, -1, scale, tree_mask, key_scale, value_scale, out)


def paged_commit(key_cache, value_cache, block_tables, prefix_lens, path, path_lens, *, key_scale=None,
                 value_scale=None) -> None:
    """Keeps accepted drafts, in place: of each sequence, the keys and values
    with index prefix_lens[b] + path[b, i] move to prefix_lens[b] + i, for i <
    path_lens[b], as if all were read before the first is written.

    prefix_lens: int32 [sequences], the keys before the drafts.  path: int32
    [sequences, up to 1024], the accepted drafts by their row in the tree, from
    the root on.  path_lens: int32 [sequences].  Entries below 0 and indices
    beyond the page table move nothing.  The sequences' lengths are then
    prefix_lens + path_lens.  At most 65535 sequences."""
    torch = _ra._torch()
    c, seqs, _, _ = _cache(key_cache, value_cache, block_tables, prefix_lens, None, key_scale, value_scale, None)
    if prefix_lens is None:
        raise TypeError("prefix_lens must be a torch.Tensor")
    device = key_cache.device
    p = _index("path", path, 2, device)
    n = _index("path_lens", path_lens, 1, device)
    if path.shape[0] != seqs or path_lens.shape[0] != seqs:
        raise ValueError(f"path and path_lens must have one row per sequence ({seqs}), got {tuple(path.shape)} and "
                         f"{tuple(path_lens.shape)}")
    if path.shape[1] > 1024:
        raise ValueError(f"path must have at most 1024 columns, got {path.shape[1]}")
    if path.numel() == 0:
        return
    _call(device, "paged_commit", _handle().rdna_paged_commit, c, c.seq_lens, p, path.stride(0), path.shape[1], n)
