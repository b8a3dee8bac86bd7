// Paged attention of few rows: the kernels of calls whose keys are in one part.
#include "paged_stream.hpp"

namespace rdna_amd {

int64_t paged_stream_cost(const PagedAttnArgs&, const PagedWork& w) {
    return paged_max_cost<kRows, kTile, 0>(w);
}

// Workers are workgroups; smallest share: a tile for every wave.
int paged_stream_attention(const PagedAttnArgs& a, PagedAttnParams& p, const PagedLaunch& l, hipStream_t stream,
                           std::string& err) {
    return paged_for_type(a, [&](auto t, auto d, auto i8) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        constexpr bool I8 = decltype(i8)::value;
        auto go = [&](auto waves) {
            constexpr int WV = decltype(waves)::value;
            const void* kernel = reinterpret_cast<const void*>(&paged_stream<T, D, I8, WV>);
            return paged_launch<kRows, kTile, 0>(
                a, kernel, 64 * WV, WV, p, l, stream, err,
                [&](dim3 grid) { hipLaunchKernelGGL((paged_stream<T, D, I8, WV>), grid, dim3(64 * WV), 0, stream, p); });
        };
        // Eight waves on a CU where there are few heads: one workgroup, which streams
        // a head's keys in one front; where there are many, two of four waves, of
        // which one begins and ends heads while the other streams.  us of eight / four,
        // 8 heads, 16 x 18432 keys, 64 x 375 to 3000 keys, 128 x 512: D = 128 192 / 200, 101 /
        // 94, 57 / 52; D = 96 190 / 192, 96 / 92, 55 / 50; int8 at D = 128, 32 x 8192 keys 115 /
        // 120, 64 x 375 to 3000 78 / 63.  At D = 64 four are faster with few heads too (16 x
        // 18432 117 / 107), but for int8 (75 / 79).
        if constexpr (D == 96 || D == 128) {
            if ((int64_t)a.seqs.B * a.Hkv < kManyHeads) {
                return go(std::integral_constant<int, 8>{});
            }
        }
        return go(std::integral_constant<int, 4>{});
    });
}

} // namespace rdna_amd
