// Host-side argument blocks of the paged operators, checked by paged_api.cpp;
// the launchers only pick kernels, size grids and enqueue.
#pragma once

#include "paged_rows.hpp"

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <string>

namespace rdna_amd {

// Largest lengths: keys a page table covers and rows of a call (sums of two
// and a window stay in 32 bits).
constexpr int64_t kPagedMaxLen = int64_t(1) << 28;

enum class PagedType : int32_t { F16 = 0, BF16 = 1 }; // of rows

// Pages of keys and values: [pages, page_size, Hkv, D] with strides in bytes
// (page, token, head), scales of int8 pages likewise in floats.
struct PagedPages {
    char* k = nullptr;
    char* v = nullptr;
    float* ks = nullptr;
    float* vs = nullptr;
    int64_t k_sp = 0, k_st = 0, k_sh = 0;
    int64_t v_sp = 0, v_st = 0, v_sh = 0;
    int64_t ks_sp = 0, ks_st = 0, ks_sh = 0;
    int64_t vs_sp = 0, vs_st = 0, vs_sh = 0;
    const int32_t* table = nullptr; // [B, width]
    int64_t table_s = 0;
    int32_t width = 0, pages = 0;
    int32_t lps = 0; // log2 of the page size
};

// Page of entry e of sequence b's table, or -1 where there is none.
#if defined(__HIP__)
__device__ __forceinline__ int32_t paged_page(const PagedPages& c, const int32_t* row, int32_t e) {
    const int32_t pg = e < c.width ? row[e] : -1;
    return (uint32_t)pg < (uint32_t)c.pages ? pg : -1;
}
#endif

struct PagedAppendArgs {
    PagedPages c;
    PagedSeqs seqs;
    PagedType type = PagedType::F16; // of the rows
    bool i8 = false;
    int32_t Hq = 0, Hkv = 0, D = 0;
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    void* q_out = nullptr;
    int64_t q_st = 0, q_sh = 0, qo_st = 0, qo_sh = 0; // bytes
    int64_t k_st = 0, k_sh = 0, v_st = 0, v_sh = 0;
    const int32_t* positions = nullptr;
    const float *cos = nullptr, *sin = nullptr;
    int32_t rot = 0; // rotated channels (0: none)
    int32_t rot_rows = 0;
    int32_t interleaved = 1;
};
int paged_append(const PagedAppendArgs& a, hipStream_t stream, std::string& err);

// Norms of an append's queries and keys (weights [D], either may be null), and
// positions of several axes: column c of the tables turns by the row's position
// rot_axes[c] of `axes`, position i of row t at positions[t * position_s + i].
enum class PagedNormType : int32_t { F16 = 0, BF16 = 1, F32 = 2 };
struct PagedNorm {
    const void *query = nullptr, *key = nullptr;
    PagedNormType type = PagedNormType::F32;
    float eps = 0.0f;
    const int32_t* rot_axes = nullptr;
    int64_t position_s = 1;
    int32_t axes = 1;
};
int paged_append_norm(const PagedAppendArgs& a, const PagedNorm& n, hipStream_t stream, std::string& err);

struct PagedCommitArgs {
    PagedPages c;
    bool i8 = false;
    int32_t B = 0, Hkv = 0, row_bytes = 0, N = 0;
    const int32_t *prefix = nullptr, *path = nullptr, *count = nullptr;
    int64_t path_s = 0;
};
int paged_commit(const PagedCommitArgs& a, hipStream_t stream, std::string& err);

// Prefixes of the sequences, in the same pages: tables [n, width], lengths [n], and
// which sequences follow each (see PagedSeqs::group).
struct PagedPrefix {
    const int32_t* table = nullptr;
    const int32_t* lens = nullptr;
    const int32_t* seqs = nullptr;
    int64_t table_s = 0;
    int32_t width = 0, n = 0; // n 0: none
};

struct PagedAttnArgs {
    PagedPages c;
    PagedSeqs seqs;
    PagedPrefix prefix;
    float* lse = nullptr; // [rows, Hq] log-sum-exp of the scores, or null
    PagedMask mask;
    PagedType type = PagedType::F16;
    bool i8 = false;
    int32_t Hq = 0, Hkv = 0, D = 0;
    int32_t max_rows_seq = 0; // rows of the longest sequence, as far as the caller knows
    const void* q = nullptr;
    void* o = nullptr;
    int64_t q_st = 0, q_sh = 0, o_st = 0, o_sh = 0; // bytes
    float scale = 1.0f;
    int32_t zero_tail = 0; // write zeros to the rows behind the last sequence
    const uint8_t* tree = nullptr; // [B, tree_n, tree_n], or null
    int64_t tree_sb = 0, tree_sr = 0;
    int32_t tree_n = 0;
};
int paged_attention(const PagedAttnArgs& a, hipStream_t stream, std::string& err);

// The attention that keys have received (paged_weights.hip): only the keys of c and seqs,
// weights [pages, page, Hkv] with strides in floats.
struct PagedWeightsArgs {
    PagedPages c;
    PagedSeqs seqs;
    PagedMask mask;
    PagedType type = PagedType::F16;
    bool i8 = false;
    int32_t Hq = 0, Hkv = 0, D = 0;
    int32_t max_rows_seq = 0;
    const void* q = nullptr;
    int64_t q_st = 0, q_sh = 0; // bytes
    const float* lse = nullptr; // [rows, Hq]
    float scale = 1.0f, decay = 1.0f;
    float* w = nullptr;
    int64_t w_sp = 0, w_st = 0, w_sh = 0;
};
int paged_key_weights(const PagedWeightsArgs& a, hipStream_t stream, std::string& err);

// The keys of the largest weights to the front (paged_evict.hip).
struct PagedEvictArgs {
    PagedPages c;
    bool i8 = false;
    int32_t B = 0, Hkv = 0, row_bytes = 0;
    const int32_t* lens = nullptr;
    int32_t budget = 0, first = 0, recent = 0;
    float* w = nullptr;
    int64_t w_sp = 0, w_st = 0, w_sh = 0;
    int32_t* new_lens = nullptr; // [B]
    int32_t* kept = nullptr;     // [B, Hkv, budget]
};
int paged_evict(const PagedEvictArgs& a, hipStream_t stream, std::string& err);

// Sets the library's thread-local error message (c_api.cpp).
void set_api_error(const char* fmt, const std::string& detail);

} // namespace rdna_amd
