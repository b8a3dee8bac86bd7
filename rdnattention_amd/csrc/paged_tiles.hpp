// Paged attention of many rows per sequence and kv head (prompts, chunks of
// them, trees of drafts): out = softmax(c Q K^T) V over the pages of each
// sequence.
//
// Bound by the matrix cores where the rows fill the tiles.  A workgroup's waves
// hold 32 rows each of one kv head's rows (token after token, the G heads of a
// token side by side, so a chunk of few tokens fills the tiles too) and share
// 64-key tiles of K and V in LDS.  A row of a tile is found through the page
// table as in paged_stream.hip, the work dealt in equal shares of key tiles
// (PagedWalk), which also splits the keys of a call of few row tiles over the chip.
//
// Step i of a wave: M(i), O += V(i - 1)^T P(i - 1) and S(i) = K(i) Q^T, one stream
// of MFMAs; then the softmax of S(i) to P(i), and one barrier.  K(i + 1) and V(i) are
// copied during step i, up to D = 128 (eight waves) the keys by waves 4-7 and the
// values by waves 0-3, into the second of two slots each.  The two waves of a SIMD drift
// apart by themselves, so that one feeds the matrix core while the other runs its
// softmax.  (Two groups of waves held half a step apart by two barriers took 2 % less
// time on B4 Hq32 Hkv8 S4096 D128 causal, 7 % more at D = 96 and on one sequence of 16
// drafts, 15 % more on int8 pages.)
//
// Q goes through LDS too (up to D = 128, where there is room), in whole lines: loaded
// straight into the MFMA layout every line was fetched several times over, 4 us of an
// item's time.  The next item's Q and first table entries are copied during an item.
#pragma once

#include "paged_launch.hpp"

namespace rdna_amd {
namespace {

constexpr int kBN = 64;
// Key tiles that an item's begin and end take the time of (about 8 us against 2.2 us).
// us with 3 / 4 / 5 / 7: B4 Hq32 Hkv8 S4096 D128 causal 681 / 666 / 675 / 676, B2 Hq16 Hkv8
// S2048 D96 74 / 74 / 78 / 78 and D256 143 / 145 / 148 / 152, int8 B2 Hq32 Hkv8 S2048 D128
// 169 / 174 / 173 / 178, 8 trees of 60 drafts 105 / 104 / 105 / 104.
constexpr int kItemCost = 4;
constexpr float kRescale = 8.0f;

// for lambdas that are called more than once: called, they would keep what they
// capture in memory
#define RDNA_INLINE __attribute__((always_inline))

template <int D, bool I8>
struct TileCfg {
    // eight waves; above D = 128 four, one per SIMD, whose O takes up to 128 registers
    static constexpr int WAVES = D <= 128 ? 8 : 4;
    static constexpr bool SPLIT = WAVES == 8; // waves 0-3 stage values, 4-7 keys
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int WAVES_PER_SIMD = D <= 32 ? 4 : (SPLIT ? 2 : 1);
    static constexpr int ROWS = 32 * WAVES;
    static constexpr bool KEEP = SPLIT && !I8; // operand addresses in registers
    static constexpr bool Q_LDS = SPLIT;
    static constexpr int DEPTH = D <= 224 ? 4 : 3; // MFMA operands in flight
    static constexpr int RB = 2 * D;
    static constexpr int KCH = D / 8;
    static constexpr int TILE_BYTES = kBN * RB;
    // four batches of 64 table entries per wave, of this item and the next; of int8 the
    // key and value scales of four tiles
    static constexpr int TAB_BYTES = I8 ? 4 * 2 * kBN * 4 : WAVES * 2048;
    static constexpr int Q_BYTES = 32 * RB; // of a wave
    static constexpr int LDS_BYTES = 4 * TILE_BYTES + TAB_BYTES + (Q_LDS ? WAVES * Q_BYTES : 0);
    static constexpr int NS = D / 16;
    static constexpr int NDT = D / 32;
    // the swizzle moves chunks within groups of SWZ: operand addresses repeat, SWZ / 2
    // steps of s and SWZ / 4 of dt further, 16 SWZ bytes on
    static constexpr int SWZ = D % 64 == 32 ? 4 : (D % 128 == 64 ? 8 : 16);
    static constexpr int KA = SWZ / 2 < NS ? SWZ / 2 : NS;
    static constexpr int VA = SWZ / 4 < NDT ? SWZ / 4 : NDT;
    static constexpr int PER = TILE_BYTES / 4096;  // 1 KB copies of a tile, of each of the four waves that have it
    static constexpr int NCH = D < 64 ? 1 : D / 64; // int8: 16-byte chunks of a tile, of each of their threads
    static_assert(LDS_BYTES <= 160 * 1024, "tiles fit the LDS");
};

template <class T, int D, bool I8>
__global__ __launch_bounds__((TileCfg<D, I8>::THREADS), (TileCfg<D, I8>::WAVES_PER_SIMD)) void paged_tiles(
    PagedAttnParams p) {
    constexpr bool JOIN = false;
    constexpr PagedJoin join = {};
#include "paged_tiles_body.inl"
}

// (At D = 32 one workgroup on a CU, not two: 128 registers do not hold the second part's
// addresses too.)
template <class T, int D, bool I8>
__global__ __launch_bounds__((TileCfg<D, I8>::THREADS), (D <= 32 ? 2 : TileCfg<D, I8>::WAVES_PER_SIMD)) void
paged_join_tiles(PagedJoinParams p) {
    constexpr bool JOIN = true;
    const PagedJoin& join = p.join;
#include "paged_tiles_body.inl"
}

// Workers are workgroups; smallest share: two key tiles.
template <bool JOIN>
int paged_tile_launch(const PagedAttnArgs& a, PagedJoinParams& p, const PagedLaunch& l, hipStream_t stream,
                      std::string& err) {
    return paged_for_type(a, [&](auto t, auto d, auto i8) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        constexpr bool I8 = decltype(i8)::value;
        using C = TileCfg<D, I8>;
        auto go = [&](auto* kernel) {
            return paged_launch<C::ROWS, kBN, kItemCost>(
                a, reinterpret_cast<const void*>(kernel), C::THREADS, 2, p, l, stream, err,
                [&](dim3 grid) { hipLaunchKernelGGL(kernel, grid, dim3(C::THREADS), 0, stream, p); });
        };
        if constexpr (JOIN) {
            return go(&paged_join_tiles<T, D, I8>);
        } else {
            return go(&paged_tiles<T, D, I8>);
        }
    });
}

} // namespace
} // namespace rdna_amd
