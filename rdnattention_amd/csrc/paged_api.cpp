// C ABI of the paged-cache operators.  Every argument that the host can see is
// checked before any HIP call, here and, the work of a whole attention call, in
// paged_merge.hip; lengths, page tables and row ranges are device memory and
// bounded where they are read (paged_rows.hpp).
#include "rdnattention_ext.h"

#include "paged_host.hpp"

#include <cmath>
#include <cstdint>
#include <exception>
#include <string>

namespace {

using rdna_amd::kPagedMaxLen;
using rdna_amd::PagedType;

bool aligned(const void* p, uintptr_t a) {
    return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}

// A stride in elements of `size` bytes over `count` of them: not negative, and all
// within 2^56 bytes, so that sums of such offsets stay in 63 bits.
bool stride_fits(int64_t stride, int64_t size, uint64_t count) {
    return stride >= 0 && stride <= (int64_t(1) << 40) && (uint64_t)(stride * size) <= (uint64_t(1) << 56) / count;
}

// ... and a multiple of 16 bytes: in bytes.
bool stride_bytes(int64_t stride, int64_t size, uint64_t count, int64_t& out) {
    if (!stride_fits(stride, size, count) || stride * size % 16 != 0) {
        return false;
    }
    out = stride * size;
    return true;
}

// For the calls that write pages: workgroups move keys and values independently.
constexpr const char* kShared = "the pages of keys and values must not be the same memory";
constexpr const char* kStrides = "strides must be multiples of 16 bytes, not negative, and stay within 2^56 bytes";

// The cache into `c` and `s`; "" or what is wrong.
std::string check_cache(const rdna_paged_cache* in, rdna_amd::PagedPages& c, bool& i8) {
    if (in == nullptr) {
        return "null cache";
    }
    if (in->dtype != RDNA_DTYPE_F16 && in->dtype != RDNA_DTYPE_BF16 && in->dtype != RDNA_DTYPE_INT8) {
        return "cache dtype must be fp16, bf16 or int8";
    }
    i8 = in->dtype == RDNA_DTYPE_INT8;
    if (in->head_dim < 32 || in->head_dim > 256 || in->head_dim % 32 != 0) {
        return "unsupported head_dim (multiples of 32 from 32 to 256)";
    }
    if (i8 && in->head_dim != 64 && in->head_dim != 128) {
        return "unsupported head_dim (only 64 and 128 with int8 pages)";
    }
    if (in->num_kv_heads == 0 || in->num_kv_heads > 65535) {
        return "num_kv_heads must be 1 to 65535";
    }
    if (in->num_seqs == 0) {
        return "empty launch grid (num_seqs must be non-zero)";
    }
    if (in->num_seqs > (1u << 24)) {
        return "num_seqs exceeds 2^24";
    }
    if (in->page_size == 0 || (in->page_size & (in->page_size - 1)) != 0 || in->page_size > (1u << 20)) {
        return "page_size must be a power of two up to 2^20";
    }
    if ((uint64_t)in->table_width * in->page_size > (uint64_t)kPagedMaxLen) {
        return "the page table covers more than 2^28 keys";
    }
    if (in->num_pages == 0 || in->num_pages > (uint32_t)INT32_MAX) {
        return "num_pages must be 1 to 2^31 - 1";
    }
    if (in->key == nullptr || in->value == nullptr || (in->block_tables == nullptr && in->table_width != 0)) {
        return "null cache pointer";
    }
    if (!aligned(in->key, 16) || !aligned(in->value, 16)) {
        return "cache base pointers must be 16-byte aligned";
    }
    if (!aligned(in->block_tables, 4) || !stride_fits(in->table_stride, 4, in->num_seqs)) {
        return "block_tables must be an aligned int32 array with a row stride that is not negative and stays within "
               "2^56 bytes";
    }
    const int64_t size = i8 ? 1 : 2;
    const uint64_t counts[3] = {in->num_pages, in->page_size, in->num_kv_heads};
    if (!stride_bytes(in->key_stride[0], size, counts[0], c.k_sp) ||
        !stride_bytes(in->key_stride[1], size, counts[1], c.k_st) ||
        !stride_bytes(in->key_stride[2], size, counts[2], c.k_sh) ||
        !stride_bytes(in->value_stride[0], size, counts[0], c.v_sp) ||
        !stride_bytes(in->value_stride[1], size, counts[1], c.v_st) ||
        !stride_bytes(in->value_stride[2], size, counts[2], c.v_sh)) {
        return std::string("cache ") + kStrides;
    }
    if (i8) {
        if (in->key_scale == nullptr || in->value_scale == nullptr) {
            return "int8 pages need key_scale and value_scale";
        }
        if (!aligned(in->key_scale, 4) || !aligned(in->value_scale, 4)) {
            return "key_scale and value_scale must be aligned float arrays";
        }
        for (int i = 0; i < 3; i++) {
            if (!stride_fits(in->key_scale_stride[i], 4, counts[i]) ||
                !stride_fits(in->value_scale_stride[i], 4, counts[i])) {
                return "scale strides must not be negative, and stay within 2^56 bytes";
            }
        }
        c.ks = in->key_scale;
        c.vs = in->value_scale;
        c.ks_sp = in->key_scale_stride[0], c.ks_st = in->key_scale_stride[1], c.ks_sh = in->key_scale_stride[2];
        c.vs_sp = in->value_scale_stride[0], c.vs_st = in->value_scale_stride[1], c.vs_sh = in->value_scale_stride[2];
    }
    c.k = static_cast<char*>(in->key);
    c.v = static_cast<char*>(in->value);
    c.table = in->block_tables;
    c.table_s = in->table_stride;
    c.width = (int32_t)in->table_width;
    c.pages = (int32_t)in->num_pages;
    c.lps = __builtin_ctz(in->page_size);
    return "";
}

std::string check_rows(const rdna_paged_cache* in, uint32_t num_rows, int32_t dtype, bool i8,
                       rdna_amd::PagedSeqs& s) {
    if (dtype != RDNA_DTYPE_F16 && dtype != RDNA_DTYPE_BF16) {
        return "rows must be fp16 or bf16";
    }
    if (!i8 && dtype != in->dtype) {
        return "rows must have the type of the pages (any with int8 pages)";
    }
    if (num_rows == 0) {
        return "empty launch grid (num_rows must be non-zero)";
    }
    if (num_rows > (uint32_t)kPagedMaxLen) {
        return "num_rows exceeds 2^28";
    }
    if (in->seq_lens == nullptr) {
        return "null seq_lens";
    }
    if (!aligned(in->seq_lens, 4) || !aligned(in->cu_seqlens, 4)) {
        return "seq_lens and cu_seqlens must be aligned int32 arrays";
    }
    if (in->cu_seqlens == nullptr && num_rows % in->num_seqs != 0) {
        return "num_rows must be a multiple of num_seqs where cu_seqlens is null";
    }
    s.lens = in->seq_lens;
    s.cu = in->cu_seqlens;
    s.B = (int32_t)in->num_seqs;
    s.rows = (int32_t)(num_rows / in->num_seqs);
    s.total = (int32_t)num_rows;
    s.max_keys = (int32_t)(in->table_width * in->page_size);
    return "";
}

// body(err): 0, or -1 with err.  No exception leaves the C ABI.
template <class F>
int32_t guarded(const char* fmt, F&& body) {
    try {
        std::string err;
        if (body(err) == 0) {
            return 0;
        }
        rdna_amd::set_api_error(fmt, err);
    } catch (const std::exception&) {
        rdna_amd::set_api_error(fmt, std::string("out of host memory"));
    }
    return -3;
}

#if defined(RDNATTENTION_NO_INT8)
bool no_int8(const rdna_paged_cache* c, const char* fmt) {
    if (c != nullptr && c->dtype == RDNA_DTYPE_INT8) {
        rdna_amd::set_api_error(fmt, "this library was built without the INT8 kernels");
        return true;
    }
    return false;
}
#endif

} // namespace

RDNA_API int32_t rdna_paged_append(const rdna_paged_cache* cache, const void* key, const void* value,
                                   int64_t key_stride_row, int64_t key_stride_h, int64_t value_stride_row,
                                   int64_t value_stride_h, uint32_t num_rows, int32_t dtype, const void* query,
                                   void* query_out, int64_t query_stride_row, int64_t query_stride_h,
                                   int64_t query_out_stride_row, int64_t query_out_stride_h, uint32_t num_heads,
                                   const int32_t* positions, const void* rot_cos, const void* rot_sin,
                                   uint32_t rot_rows, uint32_t rot_dim, int32_t rot_interleaved, void* hip_stream) {
#if defined(RDNATTENTION_NO_INT8)
    if (no_int8(cache, "Paged append unavailable: %s")) {
        return -4;
    }
#endif
    return guarded("Paged append failed: %s", [&](std::string& err) {
        rdna_amd::PagedAppendArgs a;
        err = check_cache(cache, a.c, a.i8);
        if (err.empty()) {
            err = check_rows(cache, num_rows, dtype, a.i8, a.seqs);
        }
        if (!err.empty()) {
            return -1;
        }
        a.type = dtype == RDNA_DTYPE_F16 ? PagedType::F16 : PagedType::BF16;
        a.Hkv = (int32_t)cache->num_kv_heads;
        a.D = (int32_t)cache->head_dim;
        if (key == nullptr || value == nullptr) {
            err = "null tensor pointer";
        } else if (!aligned(key, 16) || !aligned(value, 16) || !aligned(query, 16) || !aligned(query_out, 16)) {
            err = "tensor base pointers must be 16-byte aligned";
        } else if (!stride_bytes(key_stride_row, 2, num_rows, a.k_st) ||
                   !stride_bytes(key_stride_h, 2, cache->num_kv_heads, a.k_sh) ||
                   !stride_bytes(value_stride_row, 2, num_rows, a.v_st) ||
                   !stride_bytes(value_stride_h, 2, cache->num_kv_heads, a.v_sh)) {
            err = std::string("row ") + kStrides;
        } else if ((rot_cos == nullptr) != (rot_sin == nullptr)) {
            err = "pass both rot_cos and rot_sin, or neither";
        } else if (rot_cos == nullptr && (query != nullptr || positions != nullptr)) {
            err = "query and positions need rot_cos and rot_sin";
        } else if (!aligned(rot_cos, 16) || !aligned(rot_sin, 16) || !aligned(positions, 4)) {
            err = "rot_cos and rot_sin must be 16-byte aligned, positions 4-byte aligned";
        } else if (rot_cos != nullptr && (rot_dim == 0 || rot_dim % 16 != 0 || rot_dim > cache->head_dim)) {
            err = "rot_dim must be a multiple of 16 up to head_dim";
        } else if (rot_cos != nullptr && (rot_rows == 0 || rot_rows > (uint32_t)INT32_MAX)) {
            err = "rot_rows must be 1 to 2^31 - 1";
        }
        if (err.empty() && query != nullptr) {
            if (query_out == nullptr) {
                err = "query without query_out";
            } else if (num_heads == 0 || num_heads > 65535) {
                err = "num_heads must be 1 to 65535";
            } else if (!stride_bytes(query_stride_row, 2, num_rows, a.q_st) ||
                       !stride_bytes(query_stride_h, 2, num_heads, a.q_sh) ||
                       !stride_bytes(query_out_stride_row, 2, num_rows, a.qo_st) ||
                       !stride_bytes(query_out_stride_h, 2, num_heads, a.qo_sh)) {
                err = std::string("query ") + kStrides;
            } else if (query == query_out && ((num_rows > 1 && a.q_st != a.qo_st) || (num_heads > 1 && a.q_sh != a.qo_sh))) {
                err = "query_out in the place of query needs query's strides";
            }
            a.Hq = (int32_t)num_heads;
        }
        if (err.empty() &&
            (uint64_t)num_rows * (uint64_t)(2 * a.Hkv + a.Hq) * (uint64_t)(a.D / 8) > (uint64_t)INT32_MAX) {
            err = "rows x heads x head_dim exceed 2^34 channels";
        } else if (err.empty() && a.c.k == a.c.v) {
            err = kShared;
        }
        if (!err.empty()) {
            return -1;
        }
        a.k = key;
        a.v = value;
        a.q = query;
        a.q_out = query_out;
        a.positions = positions;
        a.cos = static_cast<const float*>(rot_cos);
        a.sin = static_cast<const float*>(rot_sin);
        a.rot = rot_cos != nullptr ? (int32_t)rot_dim : 0;
        a.rot_rows = (int32_t)rot_rows;
        a.interleaved = rot_interleaved != 0 ? 1 : 0;
        return rdna_amd::paged_append(a, static_cast<hipStream_t>(hip_stream), err);
    });
}

RDNA_API int32_t rdna_paged_attention(const rdna_paged_cache* cache, const void* query, void* output,
                                      int64_t query_stride_row, int64_t query_stride_h, int64_t output_stride_row,
                                      int64_t output_stride_h, uint32_t num_rows, uint32_t num_heads, int32_t dtype,
                                      uint32_t max_rows_per_seq, float scale, int32_t causal, int32_t window_size,
                                      const uint8_t* tree_mask, int64_t tree_stride_seq, int64_t tree_stride_row,
                                      uint32_t tree_n, int32_t zero_tail, void* hip_stream) {
#if defined(RDNATTENTION_NO_INT8)
    if (no_int8(cache, "Paged attention unavailable: %s")) {
        return -4;
    }
#endif
    return guarded("Paged attention failed: %s", [&](std::string& err) {
        rdna_amd::PagedAttnArgs a;
        err = check_cache(cache, a.c, a.i8);
        if (err.empty()) {
            err = check_rows(cache, num_rows, dtype, a.i8, a.seqs);
        }
        if (!err.empty()) {
            return -1;
        }
        a.type = dtype == RDNA_DTYPE_F16 ? PagedType::F16 : PagedType::BF16;
        a.Hkv = (int32_t)cache->num_kv_heads;
        a.D = (int32_t)cache->head_dim;
        if (num_heads == 0 || num_heads > 65535 || num_heads % cache->num_kv_heads != 0) {
            err = "num_heads must be a positive multiple of num_kv_heads, at most 65535";
        } else if ((uint64_t)num_rows * (num_heads / cache->num_kv_heads) > (uint64_t(1) << 30)) {
            err = "rows x heads per kv head exceed 2^30";
        } else if (query == nullptr || output == nullptr) {
            err = "null tensor pointer";
        } else if (!aligned(query, 16) || !aligned(output, 16)) {
            err = "tensor base pointers must be 16-byte aligned";
        } else if (!stride_bytes(query_stride_row, 2, num_rows, a.q_st) ||
                   !stride_bytes(query_stride_h, 2, num_heads, a.q_sh) ||
                   !stride_bytes(output_stride_row, 2, num_rows, a.o_st) ||
                   !stride_bytes(output_stride_h, 2, num_heads, a.o_sh)) {
            err = std::string("query/output ") + kStrides;
        } else if (!std::isfinite(scale)) {
            err = "scale must be finite";
        } else if (tree_mask != nullptr && (causal != 0 || window_size > 0)) {
            err = "a tree mask goes with neither causal nor window_size";
        } else if (tree_mask != nullptr &&
                   (tree_n == 0 || tree_n > (uint32_t)kPagedMaxLen ||
                    !stride_fits(tree_stride_seq, 1, cache->num_seqs) || !stride_fits(tree_stride_row, 1, tree_n))) {
            err = "tree_n must be 1 to 2^28, the mask's strides not negative and within 2^56 bytes";
        }
        if (!err.empty()) {
            return -1;
        }
        a.Hq = (int32_t)num_heads;
        a.max_rows_seq = cache->cu_seqlens == nullptr ? a.seqs.rows
                                                      : (int32_t)(max_rows_per_seq < num_rows ? max_rows_per_seq : num_rows);
        a.q = query;
        a.o = output;
        a.scale = scale;
        a.mask.causal = causal != 0 ? 1 : 0;
        // a window beyond every distance is none
        a.mask.window = window_size > 0 && window_size < (1 << 30) ? window_size : 0;
        a.zero_tail = zero_tail != 0 && cache->cu_seqlens != nullptr ? 1 : 0;
        a.tree = tree_mask;
        a.tree_sb = tree_stride_seq;
        a.tree_sr = tree_stride_row;
        a.tree_n = (int32_t)tree_n;
        return rdna_amd::paged_attention(a, static_cast<hipStream_t>(hip_stream), err);
    });
}

RDNA_API int32_t rdna_paged_commit(const rdna_paged_cache* cache, const int32_t* prefix_lens, const int32_t* path,
                                   int64_t path_stride, uint32_t path_n, const int32_t* path_lens,
                                   void* hip_stream) {
#if defined(RDNATTENTION_NO_INT8)
    if (no_int8(cache, "Paged commit unavailable: %s")) {
        return -4;
    }
#endif
    return guarded("Paged commit failed: %s", [&](std::string& err) {
        rdna_amd::PagedCommitArgs a;
        err = check_cache(cache, a.c, a.i8);
        if (!err.empty()) {
            return -1;
        }
        if (cache->num_seqs > 65535) {
            err = "num_seqs exceeds 65535";
        } else if (prefix_lens == nullptr || path == nullptr || path_lens == nullptr) {
            err = "null index pointer";
        } else if (!aligned(prefix_lens, 4) || !aligned(path, 4) || !aligned(path_lens, 4)) {
            err = "index arrays must be aligned int32 arrays";
        } else if (path_n == 0 || path_n > 1024) {
            err = "path_n must be 1 to 1024";
        } else if (!stride_fits(path_stride, 4, cache->num_seqs)) {
            err = "path_stride must not be negative, and stay within 2^56 bytes";
        } else if (a.c.k == a.c.v) {
            err = kShared;
        }
        if (!err.empty()) {
            return -1;
        }
        a.B = (int32_t)cache->num_seqs;
        a.Hkv = (int32_t)cache->num_kv_heads;
        a.row_bytes = (int32_t)cache->head_dim * (a.i8 ? 1 : 2);
        a.N = (int32_t)path_n;
        a.prefix = prefix_lens;
        a.path = path;
        a.count = path_lens;
        a.path_s = path_stride;
        return rdna_amd::paged_commit(a, static_cast<hipStream_t>(hip_stream), err);
    });
}
