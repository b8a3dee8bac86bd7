// The paged attention call: which kernels, and the merge of the items that
// several workgroups share.
#include "paged_launch.hpp"

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

namespace rdna_amd {

float softmax_log2_scale(float scale);

namespace {

constexpr int kMergeThreads = 256;
constexpr int kMergeRows = 8; // rows of a merge workgroup at most

template <bool JOIN>
struct MergeParams {
    std::conditional_t<JOIN, PagedJoinParams, PagedAttnParams> p;
    int32_t n_wg, rows, D, G; // rows of a slot
    int32_t rpb;              // rows of a workgroup
    int32_t weights;          // room for each in LDS
};

// Workgroup (w, y): rows y * rpb ... of the item that starts in worker w and
// goes on behind it, if there is one: the log-sum-exp merge of its parts, in
// fp32, rounded once.  Bound by latency: the lanes of a wave take the parts'
// weights side by side, then groups of threads the parts' O, four loads in
// flight each.  A part without a visible key (l = 0) adds nothing.
// JOIN: the rows come out as paged_row_out says.
template <class T, bool JOIN>
__global__ __launch_bounds__(kMergeThreads) void paged_merge_rows(MergeParams<JOIN> p) {
    using V4 = typename PagedVec<T>::v4;
    __shared__ PagedRowOut outs[JOIN ? kMergeRows : 1];
    __shared__ __attribute__((aligned(16))) float wgt[kPagedMaxWorkers];
    __shared__ __attribute__((aligned(16))) f4 red[kMergeThreads];
    const int w = blockIdx.x;
    const PagedRecord rec = p.p.records[w];
    const int row0 = blockIdx.y * p.rpb;
    if (row0 >= rec.rows) {
        return;
    }
    const int n = rec.w_last - w + 1;
    auto slot = [&](int s) { return (int64_t)(s == 0 ? p.n_wg + w : w + s) * p.rows; };
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    for (int r = tid >> 6; r < p.rpb && row0 + r < rec.rows; r += kMergeThreads / 64) {
        const float2* ml = reinterpret_cast<const float2*>(p.p.part_ml);
        float mx = -INFINITY;
        for (int s = lane; s < n; s += 64) {
            mx = fmaxf(mx, ml[slot(s) + row0 + r].x);
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            mx = fmaxf(mx, __shfl_xor(mx, off));
        }
        float sum = 0.0f;
        for (int s = lane; s < n; s += 64) {
            const float2 v = ml[slot(s) + row0 + r];
            const float e = part_weight(v.x, mx);
            sum += v.y * e;
            wgt[r * p.weights + s] = v.y != 0.0f ? e : -1.0f;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            sum += __shfl_xor(sum, off);
        }
        float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        if constexpr (JOIN) {
            const int row = rec.r0 + row0 + r;
            const int tok = row / p.G;
            const int64_t at = (int64_t)(rec.q0 + tok) * p.p.Hq + rec.h * p.G + row - tok * p.G;
            const PagedRowOut out = paged_row_out(p.p.join, at, mx, sum);
            inv = out.own;
            if (lane == 0) {
                outs[r] = PagedRowOut{1.0f, out.pre, out.lse2};
                paged_store_lse(p.p.join, out, at);
            }
        }
        for (int s = lane; s < n; s += 64) {
            wgt[r * p.weights + s] *= wgt[r * p.weights + s] < 0.0f ? 1.0f : inv;
        }
    }
    __syncthreads();
    const int E = p.D / 4;
    const int per = kMergeThreads / E / p.rpb; // threads per row and 4 columns
    const int e = tid % E;
    const int r = tid / E % p.rpb;
    const int sg = tid / E / p.rpb;
    const bool active = sg < per && row0 + r < rec.rows;
    f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](f4 x, float wt) { acc += wt < 0.0f ? f4{0.0f, 0.0f, 0.0f, 0.0f} : x * wt; };
    if (active) {
        const float* o = p.p.part_o + (int64_t)(row0 + r) * p.D + 4 * e;
        int s = sg;
        for (; s + 3 * per < n; s += 4 * per) {
            f4 x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[i] = *reinterpret_cast<const f4*>(o + slot(s + i * per) * p.D);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                add(x[i], wgt[r * p.weights + s + i * per]);
            }
        }
        for (; s < n; s += per) {
            add(*reinterpret_cast<const f4*>(o + slot(s) * p.D), wgt[r * p.weights + s]);
        }
    }
    if (per > 1) {
        red[tid] = acc;
        __syncthreads();
        if (sg == 0) {
            for (int i = 1; i < per && i < n; i++) {
                acc += red[(i * p.rpb + r) * E + e];
            }
        }
    }
    if (active && sg == 0) {
        const int row = rec.r0 + row0 + r;
        const int tok = row / p.G, head = rec.h * p.G + row - tok * p.G;
        char* const out = p.p.o + (int64_t)(rec.q0 + tok) * p.p.o_st + head * p.p.o_sh;
        if constexpr (JOIN) {
            paged_store<T>(p.p.join, outs[r], (int64_t)(rec.q0 + tok) * p.p.Hq + head, 4 * e, acc, out);
        } else {
            *reinterpret_cast<V4*>(out + 8 * e) = __builtin_convertvector(acc, V4);
        }
    }
}

// Workgroup x: row x % heads x of the call, all its parts (PagedParts), the prefix's and its
// own, joined as above.  Garbage in `parts` (rows that no prefix's sequences have) leads to
// no access outside the scratch.
template <class T>
__global__ __launch_bounds__(kMergeThreads) void paged_merge_parts(MergeParams<true> p) {
    using V4 = typename PagedVec<T>::v4;
    __shared__ float wgt[2 * (kPagedMaxWorkers + 1)];
    __shared__ __attribute__((aligned(16))) f4 red[kMergeThreads];
    const PagedJoin& join = p.p.join;
    const int row = blockIdx.x;
    const int t = row / join.Hq, head = row - t * join.Hq;
    if (t >= paged_rows_end(p.p.work.seqs)) {
        return;
    }
    int32_t w[2], n[2], col[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const PagedParts x = join.parts[k * join.rows + row];
        w[k] = uniform(min(max(x.w, -1), p.n_wg - 1));
        n[k] = uniform(w[k] < 0 ? 1 : min(max(x.w_last, w[k]), p.n_wg - 1) - w[k] + 1);
        col[k] = uniform(min(max(x.col, 0), p.rows - 1));
    }
    const int parts = n[0] + n[1];
    // part s: its O and (m, l)
    auto at = [&](int s, const float*& o, const float2*& ml) {
        const int k = s < n[0] ? 0 : 1;
        s -= k == 0 ? 0 : n[0];
        const int64_t r = w[k] < 0 ? (int64_t)k * join.rows + row
                                   : (int64_t)(s == 0 ? p.n_wg + w[k] : w[k] + s) * p.rows + col[k];
        o = (w[k] < 0 ? join.whole_o : p.p.part_o) + r * p.D;
        ml = reinterpret_cast<const float2*>(w[k] < 0 ? join.whole_ml : p.p.part_ml) + r;
    };
    const int tid = threadIdx.x;
    if (tid < 64) {
        const float* o;
        const float2* ml;
        float mx = -INFINITY;
        for (int s = tid; s < parts; s += 64) {
            at(s, o, ml);
            mx = fmaxf(mx, ml->y != 0.0f ? ml->x : -INFINITY);
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            mx = fmaxf(mx, __shfl_xor(mx, off));
        }
        float sum = 0.0f;
        for (int s = tid; s < parts; s += 64) {
            at(s, o, ml);
            const float2 v = *ml;
            const float e = v.y != 0.0f ? part_weight(v.x, mx) : -1.0f;
            sum += v.y != 0.0f ? v.y * e : 0.0f;
            wgt[s] = e;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            sum += __shfl_xor(sum, off);
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        for (int s = tid; s < parts; s += 64) {
            wgt[s] = wgt[s] < 0.0f ? -1.0f : wgt[s] * inv;
        }
        if (tid == 0 && join.lse != nullptr) {
            join.lse[row] = sum == 0.0f ? -INFINITY : (mx + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
        }
    }
    __syncthreads();
    const int E = p.D / 4;
    const int per = kMergeThreads / E; // parts side by side
    const int e = tid % E, sg = tid / E;
    f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (sg < per) {
        for (int s = sg; s < parts; s += per) {
            const float* o;
            const float2* ml;
            at(s, o, ml);
            const f4 x = *reinterpret_cast<const f4*>(o + 4 * e);
            acc += wgt[s] < 0.0f ? f4{0.0f, 0.0f, 0.0f, 0.0f} : x * wgt[s];
        }
    }
    red[tid] = acc;
    __syncthreads();
    if (sg == 0) {
        for (int i = 1; i < per && i < parts; i++) {
            acc += red[i * E + e];
        }
        *reinterpret_cast<V4*>(p.p.o + (int64_t)t * p.p.o_st + head * p.p.o_sh + 8 * e) =
            __builtin_convertvector(acc, V4);
    }
}

} // namespace

int paged_merge(const PagedAttnArgs& a, const PagedJoinParams& p, hipStream_t stream, std::string& err) {
    // few rows with many parts: a row per workgroup
    const int rpb =
        p.slot_rows <= 32 ? 1 : std::min({kMergeRows, kMergeThreads / (a.D / 4), kPagedMaxWorkers / p.work.n_wg});
    auto launch = [&](auto* kernel, auto join, dim3 grid) {
        const MergeParams<decltype(join)::value> m{p,        p.work.n_wg, p.slot_rows, a.D,
                                                   p.work.G, rpb,         kPagedMaxWorkers / rpb};
        hipLaunchKernelGGL(kernel, grid, dim3(kMergeThreads), 0, stream, m);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            err = hipGetErrorString(e);
            return -1;
        }
        return 0;
    };
    const bool f16 = a.type == PagedType::F16;
    if (p.join.parts != nullptr) {
        return launch(f16 ? &paged_merge_parts<_Float16> : &paged_merge_parts<__bf16>, std::true_type{},
                      dim3((uint32_t)p.join.rows));
    }
    const dim3 grid((uint32_t)p.work.n_wg, (uint32_t)((p.slot_rows + rpb - 1) / rpb));
    return p.join.any() ? launch(f16 ? &paged_merge_rows<_Float16, true> : &paged_merge_rows<__bf16, true>,
                                 std::true_type{}, grid)
                        : launch(f16 ? &paged_merge_rows<_Float16, false> : &paged_merge_rows<__bf16, false>,
                                 std::false_type{}, grid);
}

int paged_attention(const PagedAttnArgs& a, hipStream_t stream, std::string& err) {
    PagedJoinParams p{};
    p.c = a.c;
    p.work.seqs = a.seqs;
    p.work.mask = a.mask;
    p.work.Hkv = a.Hkv;
    p.work.G = a.Hq / a.Hkv;
    p.q = static_cast<const char*>(a.q);
    p.o = static_cast<char*>(a.o);
    p.q_st = a.q_st;
    p.q_sh = a.q_sh;
    p.o_st = a.o_st;
    p.o_sh = a.o_sh;
    p.scale_log2e = softmax_log2_scale(a.scale);
    p.q_sign = a.scale < 0.0f ? -1.0f : 1.0f;
    p.zero_tail = (a.zero_tail != 0 ? kTailOut : 0) | (a.lse != nullptr && a.seqs.cu != nullptr ? kTailLse : 0);
    p.Hq = a.Hq;
    p.join.Hq = a.Hq;
    p.join.D = a.D;
    p.join.lse = a.lse;
    p.tree = a.tree;
    p.tree_sb = a.tree_sb;
    p.tree_sr = a.tree_sr;
    p.tree_n = a.tree_n;

    // Rows of a sequence and kv head: up to 32 stream the keys once; more share
    // them.  Ragged sequences may be of both kinds: each launch takes its own.
    constexpr int32_t kFew = 32;
    PagedLaunch few, many;
    const bool any_many = (int64_t)a.max_rows_seq * p.work.G > kFew;
    const bool any_few = !any_many || a.seqs.cu != nullptr;
    if (any_many && any_few) {
        few.max_rows = many.min_rows = kFew;
    }
    // The prefixes' rows are those of all their sequences.  One launch has the prefixes and
    // the sequences, or the prefixes have one, by tiles, of their own before the sequences'.
    // The one saves two launches and a pass over the rows, but its row tiles are 32 rows, each
    // of which reads the prefix again, and every sequence's kv head is an item of it with a
    // begin and an end of its own: up to kItems sequences x kv heads and kUnits key tiles of all
    // the prefixes' row tiles, as far as their table's width tells.  us by tiles first / in one
    // launch, one token of each sequence, bf16, 32 heads on 8, D 128, 300 own keys, prefixes of
    // 500, 8192 and 32768 keys: 8 sequences 42 / 21, 49 / 29, 64 / 44; 32 41 / 30, 58 / 38, 75 / 106;
    // 64 54 / 43, 72 / 58, 98 / 199; 96 67 / 56, 86 / 103, 131 / 293; 128 71 / 69, 92 / 94, 142 /
    // 387; of 32 heads on 32, D 64, 32 53 / 39, 69 / 57; 128 96 / 118, 111 / 184; 32 on 1, D 128, 128
    // 66 / 42, 85 / 75; 16 on 8, D 256, 64 74 / 61, 102 / 110.  Over 600 calls of 2 to 300
    // sequences, 1 to 12 prefixes of 100 to 60000 keys, 10 to 3000 own ones, this rule is 1.2 % off
    // the faster form (geometric mean), kItems 512 without kUnits was 3.8 %.
    PagedJoinParams shared = p;
    bool together = false;
    if (a.prefix.n > 0) {
        constexpr int64_t kItems = 1024, kUnits = 32768, kSharedRows = 8192;
        const double tiles = (double)a.seqs.total * p.work.G / 32 + a.prefix.n;
        const double units = tiles * a.Hkv * ((int64_t)a.prefix.width << a.c.lps) / 32;
        together = !any_many && (int64_t)a.seqs.B * a.Hkv <= kItems && units * a.D <= (double)kUnits * 128 &&
                   (int64_t)a.seqs.total * a.Hq <= kSharedRows;
        PagedSeqs& s = shared.work.seqs;
        s.prefixes = a.prefix.n;
        s.members = a.seqs.B;
        s.prefix_lens = a.prefix.lens;
        s.prefix_keys = (int32_t)((int64_t)a.prefix.width << a.c.lps);
        s.group = a.prefix.seqs;
        s.B = a.prefix.n + a.seqs.B;
        // (with more key tiles than it can count, each launch may still count its own)
        together = together && paged_join_cost(paged_work(shared.work, PagedLaunch{})) <= INT32_MAX;
        if (!together) {
            s.B = a.prefix.n;
            shared.c.table = a.prefix.table;
            shared.c.table_s = a.prefix.table_s;
            shared.c.width = a.prefix.width;
            shared.work.mask = PagedMask{0, 0};
            shared.zero_tail = 0;
            shared.join.lse = nullptr;
        }
    }
    // refused before the first of the launches has written anything
    int64_t cost = std::max(any_many ? paged_tile_cost(a, paged_work(p.work, many)) : 0,
                            any_few ? paged_stream_cost(a, paged_work(p.work, few)) : 0);
    if (a.prefix.n > 0 && !together) {
        cost = std::max(cost, paged_tile_cost(a, paged_work(shared.work, PagedLaunch{})));
    }
    if (!together && cost > INT32_MAX) {
        err = "too many rows x heads x keys that the page table covers (up to " +
              (cost == INT64_MAX ? std::string("2^63") : std::to_string(cost)) + " key tiles, at most 2^31 - 1)";
        return -1;
    }
    StreamScratch ws(ScratchUse::PagedPrefix);
    const size_t rows = (size_t)a.seqs.total * a.Hq;
    if (together) {
        if (ws.alloc(2 * rows * ((a.D + 2) * sizeof(float) + sizeof(PagedParts)), stream, err) != 0) {
            return -1;
        }
        shared.join.parts = static_cast<PagedParts*>(ws.ptr);
        shared.join.whole_o = reinterpret_cast<float*>(shared.join.parts + 2 * rows);
        shared.join.whole_ml = shared.join.whole_o + 2 * rows * a.D;
        shared.join.prefix_table = a.prefix.table;
        shared.join.prefix_table_s = a.prefix.table_s;
        shared.join.prefix_width = a.prefix.width;
        shared.join.rows = (int32_t)rows;
        return paged_join_stream_attention(a, shared, stream, err);
    }
    if (a.prefix.n > 0) {
        if (ws.alloc(rows * (a.D + 1) * sizeof(float), stream, err) != 0) {
            return -1;
        }
        shared.join.raw_o = static_cast<float*>(ws.ptr);
        shared.join.raw_l = shared.join.raw_o + rows * a.D;
        p.join.pre_o = shared.join.raw_o;
        p.join.pre_l = shared.join.raw_l;
        if (paged_tile_attention(a, shared, PagedLaunch{}, stream, err) != 0) {
            return -1;
        }
    }
    if (any_many && paged_tile_attention(a, p, many, stream, err) != 0) {
        return -1;
    }
    return any_few ? paged_stream_attention(a, p, few, stream, err) : 0;
}

} // namespace rdna_amd
