// The writers of a paged key/value cache: new rows to their places, rotated and
// quantised on the way, and accepted drafts up behind their prefix.
//
// Both move each byte once; a large call is bound by HBM, the call of a decode
// step by its chain of dependent loads (row range, length, page, angles) and
// the launch.
#include "fa_common.hpp"
#include "paged_host.hpp"

#include <algorithm>
#include <cmath>

namespace rdna_amd {
namespace {

constexpr int kThreads = 256;

template <class T>
struct Vec8 {
    typedef T type __attribute__((ext_vector_type(8)));
};

typedef int8_t b8 __attribute__((ext_vector_type(8)));

// A thread has one 16-byte chunk (8 channels) of one row of one head; heads run
// over the keys', the values' and the queries', chunks fastest, so that a wave
// reads and writes whole cache lines.
struct AppendParams {
    PagedAppendArgs a;
    uint32_t per_row; // chunks of a token: (2 Hkv [+ Hq]) D / 8
    uint32_t chunks;  // of the call
};

// Channels 8 c .. 8 c + 7 rotated by the angles of position `pos`: (x, y) ->
// (x cos - y sin, x sin + y cos), y the neighbouring channel (interleaved) or
// the one rot / 2 away, whose chunk is `other`.  In F: fp32, or fp64 where the
// result is quantised, so that the fp16 or bf16 row before it is the nearest one
// and a value at a border of two int8 steps falls the way of the definition.
template <class T, class F>
__device__ __forceinline__ typename Vec8<T>::type rotate8(typename Vec8<T>::type x, typename Vec8<T>::type other,
                                                          const float* cos_row, const float* sin_row, int c, int half,
                                                          bool interleaved) {
    typename Vec8<T>::type y;
    if (interleaved) {
        const f4 cs = *reinterpret_cast<const f4*>(cos_row + 4 * c);
        const f4 sn = *reinterpret_cast<const f4*>(sin_row + 4 * c);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const F u = (F)(float)x[2 * i], v = (F)(float)x[2 * i + 1];
            y[2 * i] = (T)(u * (F)cs[i] - v * (F)sn[i]);
            y[2 * i + 1] = (T)(u * (F)sn[i] + v * (F)cs[i]);
        }
    } else {
        const bool second = 8 * c >= half;
        const int col = 8 * c - (second ? half : 0);
        f4 cs[2], sn[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            cs[i] = *reinterpret_cast<const f4*>(cos_row + col + 4 * i);
            sn[i] = *reinterpret_cast<const f4*>(sin_row + col + 4 * i);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const F u = (F)(float)x[e], v = (F)(float)other[e];
            const F s = (F)sn[e >> 2][e & 3];
            y[e] = (T)(u * (F)cs[e >> 2][e & 3] + v * (second ? s : -s));
        }
    }
    return y;
}

template <class T, bool I8>
__global__ __launch_bounds__(kThreads) void paged_append_rows(AppendParams p) {
    using V8 = typename Vec8<T>::type;
    const PagedAppendArgs& a = p.a;
    const uint32_t idx = blockIdx.x * kThreads + threadIdx.x;
    const bool active = idx < p.chunks;
    const uint32_t at = active ? idx : p.chunks - 1;
    const int32_t t = (int32_t)(at / p.per_row);
    const uint32_t in_row = at - (uint32_t)t * p.per_row;
    const uint32_t ch = (uint32_t)a.D / 8;
    int32_t h = (int32_t)(in_row / ch);
    const int c = (int)(in_row - (uint32_t)h * ch);
    const int which = h < a.Hkv ? 0 : h < 2 * a.Hkv ? 1 : 2; // keys, values, queries
    h -= which * a.Hkv;

    const char* src = which == 0   ? (const char*)a.k + t * a.k_st + h * a.k_sh
                      : which == 1 ? (const char*)a.v + t * a.v_st + h * a.v_sh
                                   : (const char*)a.q + t * a.q_st + h * a.q_sh;
    V8 x = *reinterpret_cast<const V8*>(src + 16 * c);
    const bool rotated = which != 1 && 8 * c < a.rot;
    const int half = a.rot / 2;
    const bool paired = rotated && !a.interleaved; // with the chunk half a rotation away
    V8 other = x;
    if (paired) {
        other = *reinterpret_cast<const V8*>(src + 16 * c + (8 * c < half ? 2 * half : -2 * half));
    }

    // the row's sequence and its place there
    int32_t b, key;
    if (a.seqs.cu == nullptr) {
        b = paged_seq_of_row(a.seqs, t);
        key = rows_clamp(a.seqs.lens[b], 0, a.seqs.max_keys) - a.seqs.rows + (t - b * a.seqs.rows);
    } else {
        // the sequence of the wave's first row: how many end at or before it, 64 at a
        // time (a binary search is a chain of loads); then on to this lane's
        const int32_t t0 = __builtin_amdgcn_readfirstlane(t);
        const int lane = threadIdx.x & 63;
        b = 0;
        for (int32_t i = 0; i < a.seqs.B; i += 64) {
            const bool ended = i + lane < a.seqs.B && a.seqs.cu[i + lane + 1] <= t0;
            b += __popcll(__builtin_amdgcn_ballot_w64(ended));
        }
        b = paged_seq_of_row(a.seqs, t, b);
        key = -1;
        if (b >= 0) {
            const PagedSeq s = paged_seq(a.seqs, b);
            key = s.len - s.n + (t - s.q0);
        }
    }
    int32_t page = -1;
    if (key >= 0 && which != 2) {
        page = paged_page(a.c, a.c.table + b * a.c.table_s, key >> a.c.lps);
    }
    if (rotated && b >= 0 && (a.positions != nullptr || key >= 0)) {
        const int32_t pos = rows_clamp(a.positions != nullptr ? a.positions[t] : key, 0, a.rot_rows - 1);
        const int64_t off = (int64_t)pos * half;
        const V8 was = x;
        if (I8 && which == 0) {
            x = rotate8<T, double>(x, other, a.cos + off, a.sin + off, c, half, a.interleaved != 0);
        } else {
            x = rotate8<T, float>(x, other, a.cos + off, a.sin + off, c, half, a.interleaved != 0);
        }
        if (which == 2 && paired) {
            other = rotate8<T, float>(other, was, a.cos + off, a.sin + off, c + half / 8, half, false);
        }
    }
    if (which == 2) {
        // The queries may be rotated in place: of two chunks that are rotated together the
        // first one's thread, which has read both, writes both.  (A head's 12, 20, 24 or 28
        // chunks straddle waves and workgroups, so the other thread may read them later.)
        char* const dst = (char*)a.q_out + t * a.qo_st + h * a.qo_sh + 16 * c;
        if (active && !(paired && 8 * c >= half)) {
            *reinterpret_cast<V8*>(dst) = x;
            if (paired) {
                *reinterpret_cast<V8*>(dst + 2 * half) = other;
            }
        }
        return;
    }
    float scale = 0.0f;
    if constexpr (I8) {
        // largest magnitude of the row: its D / 8 lanes lie side by side in one wave
        // (D 64 or 128; keys and values before queries: no lane of theirs has left)
        float mx = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = fabsf((float)x[e]);
            mx = v > mx || v != v ? v : mx;
        }
        for (int d = 1; d < (int)ch; d <<= 1) {
            const float v = __shfl_xor(mx, d);
            mx = v > mx || v != v ? v : mx;
        }
        scale = mx * (1.0f / 127.0f);
        scale = scale == 0.0f ? 1.0f : scale;
    }
    if (page < 0 || !active) {
        return;
    }
    const int32_t off = key & ((1 << a.c.lps) - 1);
    char* dst = which == 0 ? a.c.k + page * a.c.k_sp + off * a.c.k_st + h * a.c.k_sh
                           : a.c.v + page * a.c.v_sp + off * a.c.v_st + h * a.c.v_sh;
    if constexpr (I8) {
        b8 y;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            y[e] = (int8_t)fminf(fmaxf(rintf((float)x[e] / scale), -127.0f), 127.0f);
        }
        *reinterpret_cast<b8*>(dst + 8 * c) = y;
        if (c == 0) {
            float* sc = which == 0 ? a.c.ks + page * a.c.ks_sp + off * a.c.ks_st + h * a.c.ks_sh
                                   : a.c.vs + page * a.c.vs_sp + off * a.c.vs_st + h * a.c.vs_sh;
            *sc = scale;
        }
    } else {
        *reinterpret_cast<V8*>(dst + 16 * c) = x;
    }
}

// One workgroup moves a 64-byte column slice of all accepted rows of one head,
// of the keys or the values: every row is in registers before the first is
// written, so paths may name any rows in any order.  PASSES x 64 rows.
struct CommitParams {
    PagedCommitArgs a;
    int32_t slices;
};

template <int PASSES>
__global__ __launch_bounds__(kThreads) void paged_commit_rows(CommitParams p) {
    const PagedCommitArgs& a = p.a;
    const int b = blockIdx.y;
    const int slice = blockIdx.x % p.slices;
    const int hv = blockIdx.x / p.slices;
    const int h = hv >> 1;
    const bool keys = (hv & 1) == 0;
    const int32_t n = rows_clamp(a.count[b], 0, a.N);
    const int64_t prefix = a.prefix[b];
    const int32_t* table = a.c.table + b * a.c.table_s;
    const int64_t max_keys = (int64_t)a.c.width << a.c.lps;
    const int ch = threadIdx.x & 3;
    const int r0 = threadIdx.x >> 2;
    char* const base = (keys ? a.c.k + h * a.c.k_sh : a.c.v + h * a.c.v_sh) + 64 * slice + 16 * ch;
    float* const sbase = keys ? a.c.ks + h * a.c.ks_sh : a.c.vs + h * a.c.vs_sh;
    const int64_t sp = keys ? a.c.k_sp : a.c.v_sp, st = keys ? a.c.k_st : a.c.v_st;
    const int64_t ssp = keys ? a.c.ks_sp : a.c.vs_sp, sst = keys ? a.c.ks_st : a.c.vs_st;
    const bool scales = a.i8 && slice == 0 && ch == 0;
    const int32_t mask = (1 << a.c.lps) - 1;

    i4 x[PASSES];
    float sc[PASSES];
    int32_t to[PASSES]; // page of the destination, -1: nothing to move
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int r = r0 + 64 * i;
        x[i] = i4{0, 0, 0, 0};
        sc[i] = 0.0f;
        to[i] = -1;
        if (r < n) {
            const int64_t from = prefix + a.path[b * a.path_s + r], dst = prefix + r;
            if (a.path[b * a.path_s + r] >= 0 && from >= 0 && from < max_keys && dst >= 0 && dst < max_keys &&
                from != dst) {
                const int32_t pf = paged_page(a.c, table, (int32_t)(from >> a.c.lps));
                const int32_t pt = paged_page(a.c, table, (int32_t)(dst >> a.c.lps));
                if (pf >= 0 && pt >= 0) {
                    to[i] = pt;
                    const int64_t off = from & mask;
                    x[i] = *reinterpret_cast<const i4*>(base + pf * sp + off * st);
                    if (scales) {
                        sc[i] = sbase[pf * ssp + off * sst];
                    }
                }
            }
        }
    }
    // every load has returned before any wave stores
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        asm volatile("" ::"v"(x[i]), "v"(sc[i]));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        if (to[i] >= 0) {
            const int64_t off = (prefix + r0 + 64 * i) & mask;
            *reinterpret_cast<i4*>(base + to[i] * sp + off * st) = x[i];
            if (scales) {
                sbase[to[i] * ssp + off * sst] = sc[i];
            }
        }
    }
}

int launched(std::string& err) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        err = hipGetErrorString(e);
        return -1;
    }
    return 0;
}

} // namespace

int paged_append(const PagedAppendArgs& a, hipStream_t stream, std::string& err) {
    AppendParams p;
    p.a = a;
    p.per_row = (uint32_t)(2 * a.Hkv + a.Hq) * (uint32_t)(a.D / 8);
    p.chunks = (uint32_t)a.seqs.total * p.per_row;
    const dim3 grid((p.chunks + kThreads - 1) / kThreads);
    const bool f16 = a.type == PagedType::F16;
    if (a.i8) {
        auto* const kernel = f16 ? &paged_append_rows<_Float16, true> : &paged_append_rows<__bf16, true>;
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, p);
    } else {
        auto* const kernel = f16 ? &paged_append_rows<_Float16, false> : &paged_append_rows<__bf16, false>;
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, p);
    }
    return launched(err);
}

int paged_commit(const PagedCommitArgs& a, hipStream_t stream, std::string& err) {
    CommitParams p;
    p.a = a;
    p.slices = a.row_bytes / 64;
    auto* const kernel = a.N <= 64 ? &paged_commit_rows<1> : a.N <= 256 ? &paged_commit_rows<4> : &paged_commit_rows<16>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(p.slices * 2 * a.Hkv), (uint32_t)a.B), dim3(kThreads), 0, stream, p);
    return launched(err);
}

} // namespace rdna_amd
