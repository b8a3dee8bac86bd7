// Launch of the paged attention kernels: workgroups, scratch and the merge.
#pragma once

#include "fa_host.hpp"
#include "fa_internal.hpp"
#include "paged_attn.hpp"

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

namespace rdna_amd {

// Most workers of a launch (the merge's weights of one row in LDS).
constexpr int kPagedMaxWorkers = 4096;

// One launch: the sequences of more than min_rows and at most max_rows rows.
struct PagedLaunch {
    int32_t min_rows = 0;
    int32_t max_rows = INT32_MAX;
};
inline PagedWork paged_work(const PagedWork& call, const PagedLaunch& l) {
    PagedWork w = call;
    w.min_rows = l.min_rows;
    w.max_rows = l.max_rows;
    return w;
}

// The merge of the items that several workgroups share (paged_merge.hip), or of every row's
// parts where p.join.parts says where they are.
int paged_merge(const PagedAttnArgs& a, const PagedJoinParams& p, hipStream_t stream, std::string& err);

// Workers (workgroups) for at most `units` units in shares of min_units at least.
inline int paged_workgroups(int64_t resident, int64_t units, int min_units) {
    int64_t n = std::min<int64_t>({resident, kPagedMaxWorkers, (units + min_units - 1) / min_units});
    n = n >= 8 ? n / 8 * 8 : std::max<int64_t>(n, 1);
    return (int)n;
}

constexpr size_t paged_scratch_bytes(int n_wg, int rows, int D) {
    return (size_t)n_wg * (2 * (size_t)rows * (D + 2) * sizeof(float) + sizeof(PagedRecord));
}

template <int ROWS, int BN, int EXTRA, class Go>
int paged_launch(const PagedAttnArgs& a, const void* kernel, int threads, int min_units, PagedJoinParams& p,
                 const PagedLaunch& l, hipStream_t stream, std::string& err, Go&& go) {
    const int64_t resident = resident_workgroups(kernel, threads, err);
    if (resident <= 0) {
        return -1;
    }
    p.work = paged_work(p.work, l);
    p.work.min_units = min_units;
    p.work.n_wg = paged_workgroups(resident, paged_max_cost<ROWS, BN, EXTRA>(p.work), min_units);
    p.slot_rows = (int32_t)std::min<int64_t>(ROWS, (int64_t)p.work.seqs.total * p.work.G);
    const size_t bytes = paged_scratch_bytes(p.work.n_wg, p.slot_rows, a.D);
    StreamScratch ws(ScratchUse::PagedPartials);
    if (ws.alloc(bytes, stream, err) != 0) {
        return -1;
    }
    p.part_o = static_cast<float*>(ws.ptr);
    p.part_ml = p.part_o + (size_t)2 * p.work.n_wg * p.slot_rows * a.D;
    p.records = reinterpret_cast<PagedRecord*>(p.part_ml + (size_t)2 * p.work.n_wg * p.slot_rows * 2);
    {
        KernelTimerGuard timer(stream);
        go(dim3((uint32_t)p.work.n_wg));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            err = hipGetErrorString(e);
            return -1;
        }
    }
    p.zero_tail = 0; // done by the call's first launch
    return paged_merge(a, p, stream, err);
}

// f(T, integral_constant<int, D>, bool_constant<int8 pages>) for what the
// kernels are built for.
template <class T, class F>
int paged_for_dim(const PagedAttnArgs& a, F&& f) {
    if (a.i8) {
#if !defined(RDNATTENTION_NO_INT8)
        return a.D == 64 ? f(T{}, std::integral_constant<int, 64>{}, std::true_type{})
                         : f(T{}, std::integral_constant<int, 128>{}, std::true_type{});
#else
        return -1;
#endif
    }
    switch (a.D) {
    case 32: return f(T{}, std::integral_constant<int, 32>{}, std::false_type{});
    case 64: return f(T{}, std::integral_constant<int, 64>{}, std::false_type{});
    case 96: return f(T{}, std::integral_constant<int, 96>{}, std::false_type{});
    case 128: return f(T{}, std::integral_constant<int, 128>{}, std::false_type{});
    case 160: return f(T{}, std::integral_constant<int, 160>{}, std::false_type{});
    case 192: return f(T{}, std::integral_constant<int, 192>{}, std::false_type{});
    case 224: return f(T{}, std::integral_constant<int, 224>{}, std::false_type{});
    default: return f(T{}, std::integral_constant<int, 256>{}, std::false_type{});
    }
}
template <class F>
int paged_for_type(const PagedAttnArgs& a, F&& f) {
    return a.type == PagedType::F16 ? paged_for_dim<_Float16>(a, f) : paged_for_dim<__bf16>(a, f);
}

// The kernels of few rows (paged_stream.hip) and of many (paged_tiles.hip).
int paged_stream_attention(const PagedAttnArgs& a, PagedJoinParams& p, const PagedLaunch& l, hipStream_t stream,
                           std::string& err);
int paged_tile_attention(const PagedAttnArgs& a, PagedJoinParams& p, const PagedLaunch& l, hipStream_t stream,
                         std::string& err);
// ... of rows whose keys are in two parts, or with the log-sum-exp (paged_stream_out.hip,
// paged_tiles_join.hip)
int paged_out_stream_attention(const PagedAttnArgs& a, PagedJoinParams& p, const PagedLaunch& l, hipStream_t stream,
                               std::string& err);
int paged_join_tile_attention(const PagedAttnArgs& a, PagedJoinParams& p, const PagedLaunch& l, hipStream_t stream,
                              std::string& err);
// ... of few rows with their prefixes, in one launch
int paged_join_stream_attention(const PagedAttnArgs& a, PagedJoinParams& p, hipStream_t stream, std::string& err);
int64_t paged_join_cost(const PagedWork& w);
// ... and what a launch of them may cost at most (paged_max_cost).
int64_t paged_stream_cost(const PagedAttnArgs& a, const PagedWork& w);
int64_t paged_tile_cost(const PagedAttnArgs& a, const PagedWork& w);

} // namespace rdna_amd
