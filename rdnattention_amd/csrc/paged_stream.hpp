// Paged attention of few rows per sequence and kv head (single tokens, a few
// drafts): out = softmax(c Q K^T) V over the pages of each sequence.
//
// Bound by HBM: a cached byte serves only the G n rows of its head group, so
// the design keeps bytes in flight.  As in the contiguous split-K kernel
// (fa_fwd_decode.hip) a workgroup's waves work on interleaved 32-key tiles of
// their own, K and V streamed by non-temporal HBM -> LDS copies, the rows being
// the 32 columns of the MFMAs; what differs:
//
//   * a row of K or V is found through the page table: each lane takes the page
//     of one key of the tile (its entry copied to LDS in time, in the copies' own
//     order, so no wait of the compiler's drains them), leaves the row's address
//     in LDS, and every copy instruction reads the address of its lane's row back.
//     Any page size costs the same: 1 KB of LDS and about 40 instructions per tile
//   * the lengths are on the device: every workgroup derives its share of all
//     key tiles from them (PagedWalk), equal for any mix of lengths, and the
//     heads it shares with others are merged by a second launch
//   * int8 pages are copied as they are (half the bytes) and
//     widened exactly as they become MFMA operands; a key's scale multiplies its
//     scores, a value's scale its weights, in fp32 (see ValueScale), so the pages
//     cost no rounding beyond the 16-bit kernels'
#pragma once

#include "paged_attn.hpp"

#include "paged_launch.hpp"

namespace rdna_amd {
namespace {

constexpr int kRows = 32; // rows per item: columns of the MFMAs
constexpr int kTile = 32; // keys per wave tile
constexpr int kManyHeads = 512; // kv heads of all sequences: two per CU
constexpr float kRescale = 8.0f;
constexpr int kDepth = 4; // MFMA operands in flight
// paged_join_stream: what an item's begin and end cost, in key tiles of the workgroup.  One prefix
// of 8192 keys, 300 of every sequence, 8 kv heads, us at 12 / 24 / 40: 8 sequences 24.3 / 23.5 /
// 23.8, 32 39 / 35 / 46, 64 61 / 52 / 75; of 1000 keys, 64 sequences, 37 / 38 / 40.
constexpr int kJoinCost = 24;

template <int D, bool I8, int WV>
struct StreamCfg {
    // a K and a V tile of each wave, 128 D bytes (of int8 half as much), and their
    // addresses.  Above D = 128 one workgroup of four waves fills a CU (its O alone
    // takes 128 registers at 256); below, two of four waves or one of eight
    static constexpr int WAVES = WV;
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int WAVES_PER_SIMD = D <= 32 ? 4 : (D <= 64 && !I8 ? 3 : (D <= 128 ? 2 : 1));
    static constexpr int RB = I8 ? D : 2 * D; // row bytes
    static constexpr int KCH = RB / 16;
    static constexpr int TILE_BYTES = kTile * RB;
    // two batches of 64 table entries; of int8 32 key and 32 value scales; K and V row
    // addresses (32 x 8 bytes each)
    static constexpr int TAB_BYTES = 2 * 256;
    static constexpr int SCALE_BYTES = I8 ? 256 : 0;
    static constexpr int WAVE_BYTES = 2 * TILE_BYTES + TAB_BYTES + SCALE_BYTES + 2 * 256;
    static constexpr int NS = D / 16;
    static constexpr int NDT = D / 32;
    static constexpr int DMA = TILE_BYTES / 1024;
    // copies of a K tile with its scales, and of a V tile
    static constexpr int K_COPIES = DMA + (I8 ? 1 : 0);
    static constexpr int V_COPIES = DMA;
    static_assert(WAVES * WAVE_BYTES <= 160 * 1024, "tiles fit the LDS");
    // the merge: each wave's O, rows of D + 4 floats, and (m, l)
    static constexpr int MERGE_BYTES = kRows * (D + 4 + 2) * 4;
    static constexpr int LDS_BYTES = WAVES * (WAVE_BYTES > MERGE_BYTES ? WAVE_BYTES : MERGE_BYTES);
    static_assert(K_COPIES + V_COPIES + 1 < 64, "vmcnt counts them");
};

template <class T, int D, bool I8, int WV>
__global__ __launch_bounds__((StreamCfg<D, I8, WV>::THREADS), (StreamCfg<D, I8, WV>::WAVES_PER_SIMD)) void paged_stream(
    PagedAttnParams p) {
    constexpr bool JOIN = false, OUT = false;
    constexpr PagedJoin join = {};
#include "paged_stream_body.inl"
}

// A kernel of its own: asked for at the end of every item, the two ways out of a row cost
// calls without a log-sum-exp 1.1 of 9.9 us (1 x 2048 keys, 8 heads of 128).
template <class T, int D, bool I8, int WV>
__global__ __launch_bounds__((StreamCfg<D, I8, WV>::THREADS), (StreamCfg<D, I8, WV>::WAVES_PER_SIMD)) void
paged_out_stream(PagedJoinParams p) {
    constexpr bool JOIN = false, OUT = true;
    const PagedJoin& join = p.join;
#include "paged_stream_body.inl"
}

template <class T, int D, bool I8, int WV>
__global__ __launch_bounds__((StreamCfg<D, I8, WV>::THREADS), (StreamCfg<D, I8, WV>::WAVES_PER_SIMD)) void
paged_join_stream(PagedJoinParams p) {
    constexpr bool JOIN = true, OUT = false;
    const PagedJoin& join = p.join;
#include "paged_stream_body.inl"
}

// Workers are workgroups; smallest share: a tile for every wave.
template <bool OUT>
int paged_stream_launch(const PagedAttnArgs& a, PagedJoinParams& p, const PagedLaunch& l, hipStream_t stream,
                        std::string& err) {
    return paged_for_type(a, [&](auto t, auto d, auto i8) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        constexpr bool I8 = decltype(i8)::value;
        auto run = [&](auto* kernel, int waves) {
            return paged_launch<kRows, kTile, 0>(
                a, reinterpret_cast<const void*>(kernel), 64 * waves, waves, p, l, stream, err,
                [&](dim3 grid) { hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, stream, p); });
        };
        auto go = [&](auto waves) {
            constexpr int WV = decltype(waves)::value;
            if constexpr (OUT) {
                return run(&paged_out_stream<T, D, I8, WV>, WV);
            } else {
                return run(&paged_stream<T, D, I8, WV>, WV);
            }
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

} // namespace
} // namespace rdna_amd
