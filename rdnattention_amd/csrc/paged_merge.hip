// The paged attention call: which kernels, and the merge of the items that
// several workgroups share.
#include "paged_launch.hpp"

#include <algorithm>
#include <cstdint>
#include <string>

namespace rdna_amd {

float softmax_log2_scale(float scale);

namespace {

constexpr int kMergeThreads = 256;
constexpr int kMergeRows = 8; // rows of a merge workgroup at most

struct MergeParams {
    PagedAttnParams p;
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
__global__ __launch_bounds__(kMergeThreads) void paged_merge_rows(MergeParams p) {
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

} // namespace

int paged_merge(const PagedAttnArgs& a, const PagedAttnParams& p, hipStream_t stream, std::string& err) {
    MergeParams m;
    m.p = p;
    m.n_wg = p.work.n_wg;
    m.rows = p.slot_rows;
    m.D = a.D;
    m.G = p.work.G;
    // few rows with many parts: a row per workgroup
    m.rpb = p.slot_rows <= 32 ? 1 : std::min({kMergeRows, kMergeThreads / (a.D / 4), kPagedMaxWorkers / m.n_wg});
    m.weights = kPagedMaxWorkers / m.rpb;
    const dim3 grid((uint32_t)m.n_wg, (uint32_t)((m.rows + m.rpb - 1) / m.rpb));
    const bool join = p.join.any();
    auto* const kernel = a.type == PagedType::F16
                             ? (join ? &paged_merge_rows<_Float16, true> : &paged_merge_rows<_Float16, false>)
                             : (join ? &paged_merge_rows<__bf16, true> : &paged_merge_rows<__bf16, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(kMergeThreads), 0, stream, m);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        err = hipGetErrorString(e);
        return -1;
    }
    return 0;
}

int paged_attention(const PagedAttnArgs& a, hipStream_t stream, std::string& err) {
    PagedAttnParams p{};
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
    // The prefixes' rows are those of all their sequences: one launch, for all of them.
    PagedAttnParams shared = p;
    const bool shared_many = (int64_t)a.seqs.total * p.work.G > kFew;
    if (a.prefix.n > 0) {
        shared.c.table = a.prefix.table;
        shared.c.table_s = a.prefix.table_s;
        shared.c.width = a.prefix.width;
        shared.work.seqs.lens = a.prefix.lens;
        shared.work.seqs.B = a.prefix.n;
        shared.work.seqs.max_keys = (int32_t)((int64_t)a.prefix.width << a.c.lps);
        shared.work.seqs.members = a.seqs.B;
        shared.work.seqs.group = a.prefix.seqs;
        shared.work.mask = PagedMask{0, 0};
        shared.zero_tail = 0;
        shared.join.lse = nullptr;
    }
    // refused before the first of the launches has written anything
    int64_t cost = std::max(any_many ? paged_tile_cost(a, paged_work(p.work, many)) : 0,
                            any_few ? paged_stream_cost(a, paged_work(p.work, few)) : 0);
    if (a.prefix.n > 0) {
        const PagedWork w = paged_work(shared.work, PagedLaunch{});
        cost = std::max(cost, shared_many ? paged_tile_cost(a, w) : paged_stream_cost(a, w));
    }
    if (cost > INT32_MAX) {
        err = "too many rows x heads x keys that the page table covers (up to " +
              (cost == INT64_MAX ? std::string("2^63") : std::to_string(cost)) + " key tiles, at most 2^31 - 1)";
        return -1;
    }
    StreamScratch ws(ScratchUse::PagedPrefix);
    if (a.prefix.n > 0) {
        const size_t rows = (size_t)a.seqs.total * a.Hq;
        if (ws.alloc(rows * (a.D + 1) * sizeof(float), stream, err) != 0) {
            return -1;
        }
        shared.join.raw_o = static_cast<float*>(ws.ptr);
        shared.join.raw_l = shared.join.raw_o + rows * a.D;
        p.join.pre_o = shared.join.raw_o;
        p.join.pre_l = shared.join.raw_l;
        if ((shared_many ? paged_tile_attention : paged_stream_attention)(a, shared, PagedLaunch{}, stream, err) != 0) {
            return -1;
        }
    }
    if (any_many && paged_tile_attention(a, p, many, stream, err) != 0) {
        return -1;
    }
    return any_few ? paged_stream_attention(a, p, few, stream, err) : 0;
}

} // namespace rdna_amd
