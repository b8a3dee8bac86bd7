// Paged attention of few rows behind prefixes that sequences share.
#include "paged_stream.hpp"

namespace rdna_amd {

int64_t paged_join_cost(const PagedWork& w) {
    return paged_max_cost<kRows, kTile, kJoinCost>(w);
}

int paged_join_stream_attention(const PagedAttnArgs& a, PagedJoinParams& p, hipStream_t stream, std::string& err) {
    return paged_for_type(a, [&](auto t, auto d, auto i8) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        constexpr bool I8 = decltype(i8)::value;
        // 64 (32) sequences of 300 keys behind 8192, 32 heads on 8, us with 8 / 4 waves: D 32 32.0 /
        // 32.3 (21.2 / 22.5), D 64 38.4 / 38.5 (25.0 / 25.5), D 96 46.4 / 48.6 (29.5 / 28.9),
        // D 128 51.6 / 55.4 (33.7 / 34.0).  Wider heads' operands leave no registers for eight.
        constexpr int WV = D <= 128 ? 8 : 4;
        auto* const kernel = &paged_join_stream<T, D, I8, WV>;
        return paged_launch<kRows, kTile, kJoinCost>(
            a, reinterpret_cast<const void*>(kernel), 64 * WV, WV, p, PagedLaunch{}, stream, err,
            [&](dim3 grid) { hipLaunchKernelGGL(kernel, grid, dim3(64 * WV), 0, stream, p); });
    });
}

} // namespace rdna_amd
