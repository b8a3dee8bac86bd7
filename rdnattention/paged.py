"""Paged key/value caches: appending, attention, trees of drafts, commits, shared
prefixes, eviction.

Keys and values of all sequences live in pages of page_size tokens, a power of
two: ``key_cache`` and ``value_cache`` are [num_pages, page_size, kv_heads,
head_dim] (any strides of a multiple of 16 bytes with a contiguous head_dim
axis; transpose a cache kept as [num_pages, kv_heads, page_size, head_dim]), for appends and commits in
memory of their own each.  ``block_tables`` int32 [sequences, width] lists each sequence's pages in order.  The lengths
``seq_lens`` int32 [sequences] count the keys in the cache, a step's new rows
among them.  Row tensors are [rows, heads, head_dim]: without ``cu_seqlens_q``
every sequence has rows / sequences of them, with it (int32 [sequences + 1])
rows cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1 are sequence b's - it begins with
0 and never falls - and rows behind the last sequence are padding.  A sequence's n rows are its newest: row
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
import struct

import rdnattention as _ra

SUPPORTED_HEAD_DIMS_PAGED = tuple(range(32, 257, 32))

_VP, _I64, _U32, _I32, _F32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_uint32, ctypes.c_int32, ctypes.c_float

# A step's call on a short cache is as long as its host work, so the checks below
# read every property of a tensor once (70 to 160 ns each) and the cache travels
# as packed bytes (a ctypes.Structure takes 1.1 us to fill, this 0.3).

# rdna_paged_cache (include/rdnattention_ext.h): 7 pointers, 13 strides, pages,
# page_size, table_width, num_seqs, num_kv_heads, head_dim, dtype
_CACHE = struct.Struct("=7Q13q6Ii")
# rdna_paged_norm: 3 pointers, the positions' row stride, axes, eps, dtype
_NORM = struct.Struct("=3QqIfi")
_STRIDES = struct.Struct("=3q")
_F32_MAX = 3.4028234663852886e38
# rdna_paged_prefix: 3 pointers, the table's row stride, its width, prefixes
_PREFIX = struct.Struct("=3Qq2I")

_torch = _lib = _device = _raw_stream = None
_dtypes = None


def _init():
    """torch and the library, once a call needs them."""
    global _torch, _lib, _device, _raw_stream, _dtypes
    torch = _ra._torch()
    _dtypes = {torch.float16: 0, torch.bfloat16: 1, torch.int8: 2}
    _device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
        lambda i: torch.cuda.current_stream(i).cuda_stream)
    _lib = _handle()
    _torch = torch
    return torch


def _handle():
    lib = _ra._lib_handle()
    if not hasattr(lib, "rdna_paged_attention"):  # RDNATTENTION_LIB may name an older library
        raise _ra.RDNAttentionError(f"{lib._name} has no paged-cache operators: rebuild it")
    lib.rdna_paged_append.argtypes = ([_VP, _VP, _VP] + [_I64] * 4 + [_U32, _I32, _VP, _VP] + [_I64] * 4 +
                                      [_U32, _VP, _VP, _VP, _U32, _U32, _I32, _VP])
    lib.rdna_paged_append.restype = _I32
    lib.rdna_paged_attention.argtypes = ([_VP, _VP, _VP] + [_I64] * 4 + [_U32, _U32, _I32, _U32, _F32, _I32, _I32, _VP,
                                                                         _I64, _I64, _U32, _I32, _VP])
    lib.rdna_paged_attention.restype = _I32
    lib.rdna_paged_commit.argtypes = [_VP, _VP, _VP, _I64, _U32, _VP, _VP]
    lib.rdna_paged_commit.restype = _I32
    newer = {"rdna_paged_append_norm": [_VP] + lib.rdna_paged_append.argtypes,
             "rdna_paged_attention_lse": ([_VP] * 4 + [_I64] * 4 + [_U32, _U32, _I32, _U32, _F32, _I32, _I32, _I32, _VP,
                                                                    _VP]),
             "rdna_paged_key_weights": ([_VP, _VP, _I64, _I64, _U32, _U32, _I32, _U32, _VP, _F32, _I32, _I32, _F32, _VP,
                                         _VP, _VP]),
             "rdna_paged_evict": [_VP, _VP, _VP, _U32, _U32, _U32, _VP, _VP, _VP]}
    for name, args in newer.items():
        if hasattr(lib, name):  # absent from libraries built before it existed
            getattr(lib, name).argtypes, getattr(lib, name).restype = args, _I32
    return lib


def _newer(name):
    """The library's function `name`, which an older one may lack."""
    try:
        return getattr(_lib, name)
    except AttributeError:
        raise _ra.RDNAttentionError(f"{_lib._name} has no {name}: rebuild it") from None


def _index(name, t, dim, device):
    """A checked int32 tensor's (address, shape, strides)."""
    torch = _torch
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is not torch.int32:
        raise ValueError(f"{name} must be int32, got {t.dtype}")
    shape, stride = t.shape, t.stride()
    if len(shape) != dim:
        raise ValueError(f"{name} must be {dim}D, got shape {tuple(shape)}")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on the same device as key_cache")
    if stride[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name} must have contiguous rows - call .contiguous() first")
    return t.data_ptr(), shape, stride


def _cache(key_cache, value_cache, block_tables, lens, lens_name, cu_seqlens, key_scale, value_scale, rows):
    """The checked caches and sequences: (rdna_paged_cache, dtype, device,
    sequences, kv_heads, head_dim, address of lens)."""
    torch = _torch or _init()
    tensor = torch.Tensor
    if not isinstance(key_cache, tensor) or not isinstance(value_cache, tensor):
        name = "value_cache" if isinstance(key_cache, tensor) else "key_cache"
        raise TypeError(f"{name} must be a torch.Tensor")
    shape, k_stride, v_stride = key_cache.shape, key_cache.stride(), value_cache.stride()
    dtype, device = key_cache.dtype, key_cache.get_device()
    if len(shape) != 4:
        raise ValueError(f"key_cache must be 4D [pages, page_size, kv_heads, head_dim], got shape {tuple(shape)}")
    if value_cache.shape != shape or value_cache.dtype is not dtype or value_cache.get_device() != device:
        raise ValueError("value_cache must have the shape, dtype and device of key_cache")
    if k_stride[3] != 1 or v_stride[3] != 1:
        name = "value_cache" if k_stride[3] == 1 else "key_cache"
        raise ValueError(f"{name} must have a contiguous head_dim axis")
    pages, page_size, kv_heads, head_dim = shape
    code = _dtypes.get(dtype)
    ks = vs = 0
    ks_stride = vs_stride = (0, 0, 0)
    if code == 2:
        if head_dim not in _ra.SUPPORTED_HEAD_DIMS_INT8:
            raise _ra.RDNAttentionError(f"paged cache: head_dim {head_dim} not supported with int8 pages (64 and 128)")
        if key_scale is None or value_scale is None:
            raise ValueError("int8 pages need key_scale and value_scale")
        for name, t in (("key_scale", key_scale), ("value_scale", value_scale)):
            if not isinstance(t, tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if t.dtype is not torch.float32 or t.shape != shape[:3] or t.get_device() != device:
                raise ValueError(f"{name} must be a float32 tensor of shape {tuple(shape[:3])} on the device of "
                                 "key_cache")
        ks, vs, ks_stride, vs_stride = key_scale.data_ptr(), value_scale.data_ptr(), key_scale.stride(), \
            value_scale.stride()
    else:
        if code is None:
            raise ValueError(f"key_cache must be float16, bfloat16 or int8, got {dtype}")
        if key_scale is not None or value_scale is not None:
            raise ValueError("key_scale and value_scale go with int8 pages")
        if head_dim not in SUPPORTED_HEAD_DIMS_PAGED:
            raise _ra.RDNAttentionError(f"paged cache: head_dim {head_dim} not supported (multiples of 32 from 32 to 256)")
    if page_size == 0 or page_size & (page_size - 1) or page_size > 1 << 20:
        raise ValueError(f"page_size must be a power of two up to 2^20, got {page_size}")
    if pages == 0 or kv_heads == 0:
        raise ValueError(f"the caches must have pages and heads, got shape {tuple(shape)}")
    table, (seqs, width), table_stride = _index("block_tables", block_tables, 2, device)
    lens_at, lens_shape, _ = _index(lens_name, lens, 1, device)
    if lens_shape[0] != seqs:
        raise ValueError(f"{lens_name} must have one entry per row of block_tables ({seqs}), got {lens_shape[0]}")
    cu = 0
    if cu_seqlens is not None:
        cu, cu_shape, _ = _index("cu_seqlens_q", cu_seqlens, 1, device)
        if cu_shape[0] != seqs + 1:
            raise ValueError(f"cu_seqlens_q must have {seqs + 1} entries, got {cu_shape[0]}")
    elif rows and (not seqs or rows % seqs):
        raise ValueError(f"{rows} rows do not divide among {seqs} sequences (pass cu_seqlens_q)")
    packed = _CACHE.pack(key_cache.data_ptr(), value_cache.data_ptr(), ks, vs, table, lens_at, cu, k_stride[0],
                         k_stride[1], k_stride[2], v_stride[0], v_stride[1], v_stride[2], *ks_stride, *vs_stride,
                         table_stride[0], pages, page_size, width, seqs, kv_heads, head_dim, code)
    return packed, dtype, device, seqs, kv_heads, head_dim, lens_at


def _rows(name, t, rows, heads, head_dim, cache_dtype, dtype, device):
    """A row tensor [rows, heads, head_dim] (heads None: any) of a type that goes
    with the cache (dtype None), or of the given one: its (address, shape,
    strides, dtype)."""
    torch = _torch
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    shape, stride, have = t.shape, t.stride(), t.dtype
    if len(shape) != 3:
        raise ValueError(f"{name} must be 3D [rows, heads, head_dim], got shape {tuple(shape)}")
    if shape[0] != rows or shape[2] != head_dim or heads is not None and shape[1] != heads:
        raise ValueError(f"{name} must have shape ({rows}, {'any' if heads is None else heads}, {head_dim}), "
                         f"got {tuple(shape)}")
    if have is not cache_dtype and (cache_dtype is not torch.int8 or _dtypes.get(have, 2) == 2):
        raise ValueError(f"{name} must be {'float16 or bfloat16' if cache_dtype is torch.int8 else cache_dtype}, "
                         f"got {have}")
    if have is torch.int8 or dtype is not None and have is not dtype:
        raise ValueError(f"{name} must be {'float16 or bfloat16' if dtype is None else dtype}, got {have}")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on the same device as key_cache")
    if stride[2] != 1:
        raise ValueError(f"{name} must have a contiguous head_dim axis")
    return t.data_ptr(), shape, stride, have


def _call(device, what, fn, *args):
    """fn(*args, stream) on the current stream of HIP device `device`."""
    if device < 0:
        raise ValueError(f"{what}: the tensors must be on a HIP device")
    if device == _device():
        rc = fn(*args, _raw_stream(device))
    else:
        with _torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc != 0:
        raise _ra.RDNAttentionError(f"{what} failed: {_ra.last_error()}")


def _norm(query_norm, key_norm, eps, head_dim, dtype, device, rot_axes, cols, axes, stride):
    """The checked norms of an append and axes of its positions, packed."""
    torch = _torch
    code, at = 0, [0, 0]
    for i, (name, t) in enumerate((("query_norm", query_norm), ("key_norm", key_norm))):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.shape != (head_dim,) or t.get_device() != device or t.dtype is not torch.float32 and t.dtype is not dtype:
            raise ValueError(f"{name} must be a float32 or {dtype} tensor of shape ({head_dim},) on the device of "
                             f"key_cache, got {t.dtype} {tuple(t.shape)}")
        if t.stride(0) != 1:
            raise ValueError(f"{name} must be contiguous")
        if at[0] and t.dtype is not query_norm.dtype:
            raise ValueError("query_norm and key_norm must have the same dtype")
        code = 3 if t.dtype is torch.float32 else _dtypes[dtype]
        at[i] = t.data_ptr()
    if not 0.0 <= eps <= _F32_MAX:
        raise ValueError(f"norm_eps must be finite and not negative, got {eps}")
    where = 0
    if rot_axes is not None:
        if axes is None:
            raise ValueError("rot_axes needs rot_cos, rot_sin and positions")
        where, shape, _ = _index("rot_axes", rot_axes, 1, device)
        if shape[0] != cols:
            raise ValueError(f"rot_axes must have one entry per column of the tables ({cols}), got {shape[0]}")
        if not 0 < axes <= 1 << 16:
            raise ValueError(f"positions must have 1 to 65536 axes, got {axes}")
    return _NORM.pack(*at, where, stride, axes or 0, eps, code)


def paged_append(key, value, key_cache, value_cache, block_tables, seq_lens, *, cu_seqlens_q=None, query=None,
                 positions=None, rot_cos=None, rot_sin=None, rot_interleaved: bool = True, key_scale=None,
                 value_scale=None, query_norm=None, key_norm=None, norm_eps: float = 1e-6, rot_axes=None):
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

    rot_axes: int32 [rot_dim // 2], with positions [rows, axes]: column c turns by
    the row's position rot_axes[c] (time, height and width of image and video
    tokens; a number outside the axes is taken as the first or last).

    query_norm/key_norm: [head_dim] weights w (float32 or the rows' type): each
    head x of the queries or keys first becomes x w / sqrt(mean(x^2) +
    norm_eps), in the same pass and the same fp32, rounded once with the
    rotation.  With query_norm, query needs no tables.

    query: optional [rows, heads, head_dim]; returned rotated likewise, as a new
    tensor.  Padding rows, and rows without a place (a sequence shorter than
    its rows, a page outside the cache), write nothing.  Returns None without
    query."""
    torch = _torch or _init()
    if not isinstance(key, torch.Tensor):
        raise TypeError("key must be a torch.Tensor")
    rows = key.shape[0] if key.dim() else 0
    c, cache_dtype, device, seqs, kv_heads, head_dim, _ = _cache(
        key_cache, value_cache, block_tables, seq_lens, "seq_lens", cu_seqlens_q, key_scale, value_scale, rows)
    k, _, ks, dtype = _rows("key", key, rows, kv_heads, head_dim, cache_dtype, None, device)
    v, _, vs, _ = _rows("value", value, rows, kv_heads, head_dim, cache_dtype, dtype, device)
    cos = sin = pos = q = q_out = out = norm = None
    rot_rows = rot_dim = heads = 0
    axes, pos_stride = None, 1
    q_st = o_st = (0, 0)
    if rot_cos is not None and rot_sin is not None:
        for name, t in (("rot_cos", rot_cos), ("rot_sin", rot_sin)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if t.dtype is not torch.float32 or t.dim() != 2 or not t.is_contiguous() or t.get_device() != device:
                raise ValueError(f"{name} must be a contiguous 2D float32 tensor on the device of key_cache")
        table_shape = rot_cos.shape
        if table_shape != rot_sin.shape:
            raise ValueError("rot_cos and rot_sin must have the same shape")
        rot_rows, rot_dim = table_shape[0], 2 * table_shape[1]
        if rot_rows == 0 or rot_dim == 0 or rot_dim % 16 or rot_dim > head_dim:
            raise ValueError(f"rot_cos must be [positions, rot_dim // 2], rot_dim a multiple of 16 up to {head_dim}, "
                             f"got {tuple(table_shape)}")
        cos, sin = rot_cos.data_ptr(), rot_sin.data_ptr()
        if positions is not None:
            pos, pos_shape, pos_strides = _index("positions", positions, 1 if rot_axes is None else 2, device)
            if pos_shape[0] != rows:
                raise ValueError(f"positions must have one entry per row ({rows}), got {pos_shape[0]}")
            if rot_axes is not None:
                axes, pos_stride = pos_shape[1], pos_strides[0]
    elif rot_cos is not None or rot_sin is not None:
        raise ValueError("pass both rot_cos and rot_sin, or neither")
    elif query is not None and query_norm is None or positions is not None:
        raise ValueError("query and positions need rot_cos and rot_sin")
    if query is not None:
        q, (_, heads, _), q_st, _ = _rows("query", query, rows, None, head_dim, cache_dtype, dtype, device)
        out = torch.empty_like(query)
        if heads == 0:
            q = None
        else:
            q_out, o_st = out.data_ptr(), out.stride()
    elif query_norm is not None:
        raise ValueError("query_norm needs query")
    if query_norm is not None or key_norm is not None or rot_axes is not None:
        norm = _norm(query_norm if query is None or heads else None, key_norm, norm_eps, head_dim, dtype, device,
                     rot_axes, rot_dim // 2, axes, pos_stride)
    if rows == 0:
        return out
    if seqs == 0:  # nothing but padding
        return out.copy_(query) if out is not None else None
    rows_args = (k, v, ks[0], ks[1], vs[0], vs[1], rows, _dtypes[dtype], q, q_out, q_st[0], q_st[1], o_st[0], o_st[1],
                 heads, pos, cos, sin, rot_rows, rot_dim, 1 if rot_interleaved else 0)
    if norm is None:
        _call(device, "paged_append", _lib.rdna_paged_append, c, *rows_args)
    else:
        _call(device, "paged_append", _newer("rdna_paged_append_norm"), c, norm, *rows_args)
    return out


def _prefix(tables, lens, seqs, device):
    """The checked prefixes, packed."""
    table, (n, width), stride = _index("prefix_tables", tables, 2, device)
    at, shape, _ = _index("prefix_lens", lens, 1, device)
    if n == 0 or shape[0] != n:
        raise ValueError(f"prefix_lens must have one entry per row of prefix_tables ({n}, at least one), got "
                         f"{shape[0]}")
    of = 0
    if seqs is not None:
        of, shape, _ = _index("prefix_seqs", seqs, 1, device)
        if shape[0] != n + 1:
            raise ValueError(f"prefix_seqs must have {n + 1} entries, got {shape[0]}")
    elif n != 1:
        raise ValueError(f"{n} prefixes need prefix_seqs")
    return _PREFIX.pack(table, at, of, stride[0], width, n)


def _attend(what, query, key_cache, value_cache, block_tables, seq_lens, cu_seqlens_q, max_seqlen_q, is_causal,
            window_size, scale, tree_mask, key_scale, value_scale, out, return_lse=False, prefix=None):
    torch = _torch or _init()
    if not isinstance(query, torch.Tensor):
        raise TypeError("query must be a torch.Tensor")
    rows = query.shape[0] if query.dim() else 0
    c, cache_dtype, device, seqs, kv_heads, head_dim, _ = _cache(
        key_cache, value_cache, block_tables, seq_lens, "seq_lens", cu_seqlens_q, key_scale, value_scale, rows)
    q, (_, heads, _), qs, dtype = _rows("query", query, rows, None, head_dim, cache_dtype, None, device)
    if heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a multiple of kv heads ({kv_heads})")
    tree, t_sb, t_sr, t_n = None, 0, 0, 0
    if tree_mask is not None:
        if not isinstance(tree_mask, torch.Tensor):
            raise TypeError("tree_mask must be a torch.Tensor")
        shape, stride = tree_mask.shape, tree_mask.stride()
        if tree_mask.dtype is not torch.bool or len(shape) != 3 or tree_mask.get_device() != device:
            raise ValueError("tree_mask must be a 3D bool tensor on the device of key_cache")
        t_n = shape[1]
        if shape[0] != seqs or shape[2] != t_n:
            raise ValueError(f"tree_mask must have shape [{seqs}, drafts, drafts], got {tuple(shape)}")
        if cu_seqlens_q is None and seqs and rows // seqs > t_n:
            raise ValueError(f"tree_mask covers {t_n} drafts, the call has {rows // seqs} per sequence")
        if t_n == 0 and seqs:
            raise ValueError("tree_mask covers no draft")
        if t_n > 1 and stride[2] != 1:
            raise ValueError("tree_mask must have contiguous rows - call .contiguous() first")
        tree, t_sb, t_sr = tree_mask.data_ptr(), stride[0], stride[1]
    if out is None:
        zero_tail = 1
        out = torch.empty_like(query)
        o, os_ = out.data_ptr(), out.stride()
    else:
        zero_tail = 0
        o, _, os_, _ = _rows("out", out, rows, heads, head_dim, cache_dtype, dtype, device)
    if prefix is not None:
        prefix = _prefix(*prefix, device)
    lse = torch.empty(rows, heads, dtype=torch.float32, device=query.device) if return_lse else None
    if rows == 0 or heads == 0:
        return (out, lse) if return_lse else out
    if seqs == 0:  # nothing but padding
        out = out.zero_() if zero_tail else out
        return (out, lse.fill_(float("-inf"))) if return_lse else out
    most = rows if max_seqlen_q is None else max(0, min(rows, int(max_seqlen_q)))
    args = (q, o, qs[0], qs[1], os_[0], os_[1], rows, heads, _dtypes[dtype], most,
            head_dim ** -0.5 if scale is None else float(scale), 1 if is_causal else 0,
            max(-1, min(int(window_size), 2 ** 31 - 1)))
    if return_lse or prefix is not None:
        _call(device, what, _newer("rdna_paged_attention_lse"), c, prefix, *args, zero_tail,
              lse.data_ptr() if return_lse else None)
        return (out, lse) if return_lse else out
    _call(device, what, _lib.rdna_paged_attention, c, *args, tree, t_sb, t_sr, t_n, zero_tail)
    return out


def paged_attention(query, key_cache, value_cache, block_tables, seq_lens, *, cu_seqlens_q=None, max_seqlen_q=None,
                    is_causal: bool = True, window_size: int = -1, scale=None, key_scale=None, value_scale=None,
                    out=None, return_lse: bool = False):
    """Attention of each sequence's newest rows over its pages: single tokens,
    chunks of a prompt, whole prompts, or all of them in one ragged batch.

    query: float16 or bfloat16 [rows, heads, head_dim], a multiple of the
    caches' heads, the rows' keys already appended.  is_causal and window_size
    as in flash_attn, aligned to the end of the keys; a row that sees no key
    comes out as zeros.  scale defaults to 1/sqrt(head_dim).  max_seqlen_q: most
    rows of any sequence (with cu_seqlens_q; default: all rows) - it picks
    kernels, which round in other places, and decides nothing else.  Keys and values
    that some row of a sequence sees should be finite: weights of zero are
    multiplied too, so others may reach rows that do not see them.

    out: optional tensor like query to write to, whose padding rows stay as they
    are; a new tensor's are zeros.  Returns the output, with return_lse (output,
    lse): float32 [rows, heads], the logarithm of the sum of exp(score) over the
    keys that the row sees, -inf where it sees none and of padding rows.  The output
    may differ in its last bit from the call without."""
    return _attend("paged_attention", query, key_cache, value_cache, block_tables, seq_lens, cu_seqlens_q, max_seqlen_q,
                   is_causal, window_size, scale, None, key_scale, value_scale, out, return_lse)


def paged_prefix_attention(query, key_cache, value_cache, prefix_tables, prefix_lens, block_tables, seq_lens, *,
                           prefix_seqs=None, cu_seqlens_q=None, max_seqlen_q=None, is_causal: bool = True, scale=None,
                           key_scale=None, value_scale=None, out=None, return_lse: bool = False):
    """Attention of sequences that share prefixes: an instruction text, a document,
    the prompt of several samples.

    Row i of prefix_tables (int32 [prefixes, width]) lists the pages of a prefix,
    prefix_lens (int32 [prefixes]) counts its keys, and sequences prefix_seqs[i] ..
    prefix_seqs[i + 1] - 1 follow it: prefix_seqs (int32 [prefixes + 1]) begins with
    0, never falls and ends with the number of sequences; without it there is one
    prefix, of all of them.  block_tables and seq_lens are of the sequences' own
    keys alone, all else as in paged_attention: every row sees the whole prefix,
    and its own keys as is_causal says.  Each prefix is read once for all of its
    sequences.  A length of 0 is no prefix.  (A position in the text is the
    prefix's length more than the row's index: paged_append's positions.)  Calls of
    many rows take scratch of rows * heads * (head_dim + 1) float32."""
    return _attend("paged_prefix_attention", query, key_cache, value_cache, block_tables, seq_lens, cu_seqlens_q,
                   max_seqlen_q, is_causal, -1, scale, None, key_scale, value_scale, out, return_lse,
                   (prefix_tables, prefix_lens, prefix_seqs))


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
    c, _, device, seqs, _, _, prefix = _cache(key_cache, value_cache, block_tables, prefix_lens, "prefix_lens", None,
                                              key_scale, value_scale, None)
    p, path_shape, path_stride = _index("path", path, 2, device)
    n, n_shape, _ = _index("path_lens", path_lens, 1, device)
    if path_shape[0] != seqs or n_shape[0] != seqs:
        raise ValueError(f"path and path_lens must have one row per sequence ({seqs}), got {tuple(path_shape)} and "
                         f"{tuple(n_shape)}")
    if path_shape[1] > 1024:
        raise ValueError(f"path must have at most 1024 columns, got {path_shape[1]}")
    if path_shape[1] == 0 or seqs == 0:
        return
    _call(device, "paged_commit", _lib.rdna_paged_commit, c, prefix, p, path_stride[0], path_shape[1], n)


def _key_weights(t, shape, device):
    """The checked weights' address and packed strides."""
    if not isinstance(t, _torch.Tensor):
        raise TypeError("key_weights must be a torch.Tensor")
    if t.dtype is not _torch.float32 or t.shape != shape or t.get_device() != device:
        raise ValueError(f"key_weights must be a float32 tensor of shape {tuple(shape)} on the device of key_cache, "
                         f"got {t.dtype} {tuple(t.shape)}")
    if any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
        raise ValueError("key_weights must not be expanded: every weight has memory of its own")
    return t.data_ptr(), _STRIDES.pack(*t.stride())


def paged_key_weights(query, lse, key_cache, block_tables, seq_lens, key_weights, *, cu_seqlens_q=None,
                      max_seqlen_q=None, is_causal: bool = True, window_size: int = -1, scale=None, key_scale=None,
                      decay: float = 1.0) -> None:
    """Adds the attention that each cached key has received from a step's rows to
    its weight, in place:

        w = (decay * w, or 0 for the rows' own keys) + sum of exp(score - lse)

    over the rows and the heads that share the key's kv head.  query, is_causal,
    window_size and scale as the step's paged_attention or paged_prefix_attention
    had them, lse (float32 [rows, heads]) as it returned it; behind a prefix the
    weights are of the sequences' own keys.  key_weights: float32 [num_pages,
    page_size, kv_heads], any strides but those of an expanded tensor.  The rows' own keys begin at 0, so weights
    of pages that are handed out again need no clearing.  decay: at least 0; with
    0 old weights are not read.  Sequences without rows are left as they are.  No page
    may belong to two sequences with rows: the sums of one of them could be lost.
    Returns None."""
    torch = _torch or _init()
    if not isinstance(query, torch.Tensor):
        raise TypeError("query must be a torch.Tensor")
    rows = query.shape[0] if query.dim() else 0
    c, cache_dtype, device, seqs, kv_heads, head_dim, _ = _cache(
        key_cache, key_cache, block_tables, seq_lens, "seq_lens", cu_seqlens_q, key_scale, key_scale, rows)
    q, (_, heads, _), qs, dtype = _rows("query", query, rows, None, head_dim, cache_dtype, None, device)
    if heads % kv_heads:
        raise ValueError(f"query heads ({heads}) must be a multiple of kv heads ({kv_heads})")
    if not isinstance(lse, torch.Tensor):
        raise TypeError("lse must be a torch.Tensor")
    if lse.dtype is not torch.float32 or lse.shape != (rows, heads) or lse.get_device() != device:
        raise ValueError(f"lse must be a float32 tensor of shape ({rows}, {heads}) on the device of key_cache, got "
                         f"{lse.dtype} {tuple(lse.shape)}")
    if not lse.is_contiguous():
        raise ValueError("lse must be contiguous")
    w, w_stride = _key_weights(key_weights, key_cache.shape[:3], device)
    if not 0.0 <= decay <= _F32_MAX:
        raise ValueError(f"decay must be finite and not negative, got {decay}")
    if rows == 0 or heads == 0 or seqs == 0:
        return
    most = rows if max_seqlen_q is None else max(0, min(rows, int(max_seqlen_q)))
    _call(device, "paged_key_weights", _newer("rdna_paged_key_weights"), c, q, qs[0], qs[1], rows, heads,
          _dtypes[dtype], most, lse.data_ptr(), head_dim ** -0.5 if scale is None else float(scale), 1 if is_causal else 0,
          max(-1, min(int(window_size), 2 ** 31 - 1)), decay, w, w_stride)


def paged_evict(key_cache, value_cache, block_tables, seq_lens, key_weights, budget, *, first: int = 0,
                recent: int = 0, key_scale=None, value_scale=None):
    """Keeps `budget` keys of every sequence that has more, in place, each kv head
    its own: the `first` first keys, the `recent` newest ones, and of those
    between the ones of the largest key_weights (of equal ones those in front; NaN
    is below all).  They move up to the front of the sequence in their order, with
    their values, scales and weights; pages behind the new lengths are free.  No page may
    belong to two sequences (a shared prefix is no part of these tables).

    Returns (lens, kept): int32 [sequences], the lengths after it, min(length,
    budget) - seq_lens itself is left as it is; and int32 [sequences, kv_heads,
    budget], which keys they were, -1 behind the last.  Later rows are appended
    behind the new lengths with the positions of the text (paged_append's
    positions).  At most 65535 sequences."""
    torch = _torch or _init()
    c, _, device, seqs, kv_heads, _, _ = _cache(key_cache, value_cache, block_tables, seq_lens, "seq_lens", None,
                                                key_scale, value_scale, None)
    w, w_stride = _key_weights(key_weights, key_cache.shape[:3], device)
    budget, first, recent = int(budget), int(first), int(recent)
    if not 0 < budget <= 1 << 28:
        raise ValueError(f"budget must be 1 to 2^28, got {budget}")
    if first < 0 or recent < 0 or first + recent > budget:
        raise ValueError(f"first ({first}) and recent ({recent}) must not be negative, nor exceed budget ({budget}) "
                         "together")
    lens = torch.empty(seqs, dtype=torch.int32, device=key_cache.device)
    kept = torch.empty(seqs, kv_heads, budget, dtype=torch.int32, device=key_cache.device)
    if seqs:
        _call(device, "paged_evict", _newer("rdna_paged_evict"), c, w, w_stride, budget, first, recent, lens.data_ptr(),
              kept.data_ptr())
    return lens, kept
