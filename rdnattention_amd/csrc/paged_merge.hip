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
    const float* part_o;
    const float* part_ml;
    const PagedRecord* records;
    char* o;
    int64_t o_st, o_sh;
    int32_t n_wg, rows, D, G; // rows of a slot
    int32_t rpb;              // rows of a workgroup
    int32_t weights;          // room for each in LDS
};

// Workgroup (w, y): rows y * rpb ... of the item that starts in worker w and
// goes on behind it, if there is one: the log-sum-exp merge of its parts, in
// fp32, rounded once.  Bound by latency: the lanes of a wave take the parts'
// weights side by side, then groups of threads the parts' O, four loads in
// flight each.  A part without a visible key (l = 0) adds nothing.
template <class T>
__global__ __launch_bounds__(kMergeThreads) void paged_merge_rows(MergeParams p) {
    using V4 = typename PagedVec<T>::v4;
    __shared__ __attribute__((aligned(16))) float wgt[kPagedMaxWorkers];
    __shared__ __attribute__((aligned(16))) f4 red[kMergeThreads];
    const int w = blockIdx.x;
    const PagedRecord rec = p.records[w];
    const int row0 = blockIdx.y * p.rpb;
    if (row0 >= rec.rows) {
        return;
    }
    const int n = rec.w_last - w + 1;
    auto slot = [&](int s) { return (int64_t)(s == 0 ? p.n_wg + w : w + s) * p.rows; };
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    for (int r = tid >> 6; r < p.rpb && row0 + r < rec.rows; r += kMergeThreads / 64) {
        const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
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
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
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
        const float* o = p.part_o + (int64_t)(row0 + r) * p.D + 4 * e;
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
        const int tok = row / p.G;
        *reinterpret_cast<V4*>(p.o + (int64_t)(rec.q0 + tok) * p.o_st + (rec.h * p.G + row - tok * p.G) * p.o_sh +
                               8 * e) = __builtin_convertvector(acc, V4);
    }
}

} // namespace

int paged_merge(const PagedAttnArgs& a, const PagedAttnParams& p, hipStream_t stream, std::string& err) {
    MergeParams m;
    m.part_o = p.part_o;
    m.part_ml = p.part_ml;
    m.records = p.records;
    m.o = p.o;
    m.o_st = p.o_st;
    m.o_sh = p.o_sh;
    m.n_wg = p.work.n_wg;
    m.rows = p.slot_rows;
    m.D = a.D;
    m.G = p.work.G;
    // few rows with many parts: a row per workgroup
    m.rpb = p.slot_rows <= 32 ? 1 : std::min({kMergeRows, kMergeThreads / (a.D / 4), kPagedMaxWorkers / m.n_wg});
    m.weights = kPagedMaxWorkers / m.rpb;
    const dim3 grid((uint32_t)m.n_wg, (uint32_t)((m.rows + m.rpb - 1) / m.rpb));
    if (a.type == PagedType::F16) {
        hipLaunchKernelGGL(paged_merge_rows<_Float16>, grid, dim3(kMergeThreads), 0, stream, m);
    } else {
        hipLaunchKernelGGL(paged_merge_rows<__bf16>, grid, dim3(kMergeThreads), 0, stream, m);
    }
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
    p.zero_tail = a.zero_tail;
    p.Hq = a.Hq;
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
    // refused before the first of two launches has written anything
    const int64_t cost = std::max(any_many ? paged_tile_cost(a, paged_work(p.work, many)) : 0,
                                  any_few ? paged_stream_cost(a, paged_work(p.work, few)) : 0);
    if (cost > INT32_MAX) {
        err = "too many rows x heads x keys that the page table covers (up to " +
              (cost == INT64_MAX ? std::string("2^63") : std::to_string(cost)) + " key tiles, at most 2^31 - 1)";
        return -1;
    }
    if (any_many && paged_tile_attention(a, p, many, stream, err) != 0) {
        return -1;
    }
    return any_few ? paged_stream_attention(a, p, few, stream, err) : 0;
}

} // namespace rdna_amd
