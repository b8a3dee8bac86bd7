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
//     of one key of the tile (its entry copied to LDS one tile ahead, in the
//     copies' own order, so no wait of the compiler's drains them), leaves the
//     row's address in LDS, and every copy instruction reads the address of its
//     lane's row back.  Any page size costs the same: 0.75 KB of LDS and about 40
//     instructions per tile
//   * the lengths are on the device: every workgroup derives its share of all
//     key tiles from them (PagedWalk), equal for any mix of lengths, and the
//     heads it shares with others are merged by a second launch
//   * int8 pages are copied as they are (half the bytes, two tiles deep) and
//     widened exactly as they become MFMA operands; a key's scale multiplies its
//     scores, a value's scale its weights, in fp32 (see ValueScale), so the pages
//     cost no rounding beyond the 16-bit kernels'
#include "paged_attn.hpp"

#include "paged_launch.hpp"

namespace rdna_amd {
namespace {

constexpr int kRows = 32; // rows per item: columns of the MFMAs
constexpr int kTile = 32; // keys per wave tile
constexpr float kRescale = 8.0f;

template <int D, bool I8>
struct StreamCfg {
    // K and V tiles of each wave, 128 D bytes (of int8: two of each, as much), and
    // their addresses: eight waves up to D = 128, then four (one wave per SIMD, whose
    // O alone takes 128 registers at 256)
    static constexpr int WAVES = D <= 128 ? 8 : 4;
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int WAVES_PER_SIMD = D <= 32 ? 4 : (D <= 64 && !I8 ? 3 : (WAVES > 4 ? 2 : 1));
    static constexpr int SLOTS = I8 ? 2 : 1;
    static constexpr int RB = I8 ? D : 2 * D; // row bytes
    static constexpr int KCH = RB / 16;
    static constexpr int TILE_BYTES = kTile * RB;
    // per slot 64 table entries (and of int8 32 key and 32 value scales); K and V
    // row addresses (32 x 8 bytes each)
    static constexpr int TAB_BYTES = 256 * SLOTS;
    static constexpr int SCALE_BYTES = I8 ? 256 * SLOTS : 0;
    static constexpr int WAVE_BYTES = 2 * SLOTS * TILE_BYTES + TAB_BYTES + SCALE_BYTES + 2 * 256;
    static constexpr int NS = D / 16;
    static constexpr int NDT = D / 32;
    static constexpr int DMA = TILE_BYTES / 1024;
    // copies of a K tile with its scales and a later tile's entries, and of a V tile
    static constexpr int K_COPIES = DMA + (I8 ? 1 : 0) + 1;
    static constexpr int V_COPIES = DMA;
    static_assert(WAVES * WAVE_BYTES <= 160 * 1024, "tiles fit the LDS");
    static_assert(finish_lds_bytes(D, WAVES) <= WAVES * WAVE_BYTES, "the merge reuses the tile area");
    static_assert(SLOTS * (K_COPIES + V_COPIES) < 64, "vmcnt counts them");
};

// 16-byte chunk swizzle of row r of an int8 tile: rows of 64 or 128 bytes, the 64
// banks 256, so rows r and r + 4 or r + 2 start in the same bank
template <int D>
__device__ __forceinline__ int swz8(int r) {
    return D == 64 ? (r >> 2) & 3 : (r >> 1) & 7;
}

template <class T, int D, bool I8>
__global__ __launch_bounds__((StreamCfg<D, I8>::THREADS), (StreamCfg<D, I8>::WAVES_PER_SIMD)) void paged_stream(
    PagedAttnParams p) {
    using C = StreamCfg<D, I8>;
    using V8 = typename PagedVec<T>::v8;
    using V4 = typename PagedVec<T>::v4;
    // weights and values meet in P: int8 values are exact in fp16, whose weights
    // round finer than bf16's
    using P = std::conditional_t<I8, _Float16, T>;
    using P8 = typename PagedVec<P>::v8;
    __shared__ __attribute__((aligned(16))) char dsm[C::WAVES * C::WAVE_BYTES];

    const int tid = threadIdx.x;
    const int wave = uniform(tid >> 6);
    const int lane = tid & 63;
    const int l32 = lane & 31;
    const int g = lane >> 5;
    // slot i: K tile, V tile; then table entries, scales, row addresses
    char* const wsm = dsm + wave * C::WAVE_BYTES;
    char* const aux = wsm + 2 * C::SLOTS * C::TILE_BYTES;
    const uint32_t lds_w = (uint32_t)reinterpret_cast<uintptr_t>(wsm);
    const uint32_t lds_aux = lds_w + 2 * C::SLOTS * C::TILE_BYTES;
    uint64_t* const krow_at = reinterpret_cast<uint64_t*>(aux + C::TAB_BYTES + C::SCALE_BYTES);
    uint64_t* const vrow_at = krow_at + kTile;

    if (p.zero_tail != 0) {
        zero_tail_rows<D>(p);
    }
    PagedRecord rec = {};
    PagedWalk<kRows, kTile> walk(p.work);

    // lane i of copy j writes LDS bytes 1024 j + 16 i of the tile: stored chunk n %
    // KCH of row n / KCH, n = 64 j + i, which holds chunk (n % KCH) ^ swz(row)
    uint32_t src[C::DMA]; // row * 8 | chunk byte << 16
#pragma unroll
    for (int j = 0; j < C::DMA; j++) {
        const int n = 64 * j + lane;
        const int r = n / C::KCH;
        src[j] = (uint32_t)(r * 8) | (uint32_t)(((n - r * C::KCH) ^ (I8 ? swz8<D>(r) : paged_swz<D>(r))) * 16) << 16;
    }
    const uint32_t page_mask = (1u << p.c.lps) - 1u;

    while (walk.more()) {
        const PagedSeq seq = walk.seq;
        const PagedTile item = walk.tile;
        const bool whole = walk.whole();
        const int h = walk.h;
        const int G = p.work.G;
        const int r0 = walk.rt * kRows;
        const int n_rows = min(kRows, seq.n * G - r0);

        // column l32 <-> row r0 + l32: token (r0 + l32) / G, head h G + (r0 + l32) % G
        const bool col_valid = l32 < n_rows;
        const int tok = col_valid ? (r0 + l32) / G : r0 / G;
        const int head = h * G + (col_valid ? r0 + l32 - tok * G : 0);
        int row_lo, row_hi;
        row_key_bounds(paged_mask(p.work.mask, seq), tok, row_lo, row_hi);
        if (!col_valid) {
            row_lo = 1;
            row_hi = 0;
        }
        const int prefix = seq.len - seq.n;
        const uint8_t* tree_row = nullptr;
        int tree_n = 0;
        if (p.tree != nullptr) {
            tree_n = tok < p.tree_n ? min(p.tree_n, seq.n) : 0;
            tree_row = p.tree + walk.b * p.tree_sb + (tok < p.tree_n ? tok : 0) * p.tree_sr;
        }

        const int t0 = item.first + walk.at;
        const int nt = item.hi >= item.lo ? walk.count() : 0;
        const int my_tiles = nt > wave ? (nt - wave + C::WAVES - 1) / C::WAVES : 0;
        auto tile_key = [&](int j) { return (t0 + wave + C::WAVES * j) * kTile; };
        const char* const kbase = p.c.k + h * p.c.k_sh;
        const char* const vbase = p.c.v + h * p.c.v_sh;
        const int32_t* const table = p.c.table + walk.b * p.c.table_s;

        i32x4_t tab_rsrc = make_rsrc_v(table, (uint32_t)p.c.width * 4u);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            tab_rsrc[e] = uniform(tab_rsrc[e]);
        }
        // slot of tile j
        auto slot_of = [&](int j) { return C::SLOTS == 1 ? 0 : j & (C::SLOTS - 1); };
        auto issue_tab = [&](int j) {
            dma_load4(tab_rsrc, (uint32_t)((tile_key(j) + l32) >> p.c.lps) * 4u, lds_aux + 256 * slot_of(j));
        };
        uint64_t v_next = 0; // address of V row l32 of the tile whose K was issued last
        // K tile j, its scales, and then (its own entries read) the entries of the
        // tile that follows it in its slot
        auto issue_k = [&](int j) {
            const int key = tile_key(j) + l32;
            const uint32_t pg = reinterpret_cast<const uint32_t*>(aux)[64 * slot_of(j) + lane];
            const bool seen = key >= item.lo && key <= item.hi;
            const uint64_t pe = pg < (uint32_t)p.c.pages ? pg : 0u;
            const uint64_t off = (uint32_t)key & page_mask;
            const uint64_t zero = reinterpret_cast<uint64_t>(kPagedZeroRow);
            const uint64_t ka = reinterpret_cast<uint64_t>(kbase) + pe * (uint64_t)p.c.k_sp + off * (uint64_t)p.c.k_st;
            const uint64_t va = reinterpret_cast<uint64_t>(vbase) + pe * (uint64_t)p.c.v_sp + off * (uint64_t)p.c.v_st;
            v_next = seen ? va : zero;
            if (g == 0) {
                krow_at[l32] = seen ? ka : zero;
            }
            const uint32_t lds = lds_w + (uint32_t)slot_of(j) * (2 * C::TILE_BYTES);
#pragma unroll
            for (int d = 0; d < C::DMA; d++) {
                const uint64_t row = *reinterpret_cast<const uint64_t*>(reinterpret_cast<const char*>(krow_at) +
                                                                        (src[d] & 0xffffu));
                dma_gather16_nt(row + (src[d] >> 16), lds + 1024 * d);
            }
            if constexpr (I8) { // lanes 0 - 31: the keys', 32 - 63: the values'
                const uint64_t ks = reinterpret_cast<uint64_t>(p.c.ks) +
                                    4 * (pe * (uint64_t)p.c.ks_sp + off * (uint64_t)p.c.ks_st + h * (uint64_t)p.c.ks_sh);
                const uint64_t vs = reinterpret_cast<uint64_t>(p.c.vs) +
                                    4 * (pe * (uint64_t)p.c.vs_sp + off * (uint64_t)p.c.vs_st + h * (uint64_t)p.c.vs_sh);
                dma_gather4(seen ? (g == 0 ? ks : vs) : zero, lds_aux + C::TAB_BYTES + 256 * slot_of(j));
            }
            __builtin_amdgcn_s_waitcnt(waitcnt_lgkm(0)); // the entries are read
            issue_tab(j + C::SLOTS);
        };
        auto issue_v = [&](int j) {
            if (g == 0) {
                vrow_at[l32] = v_next;
            }
            const uint32_t lds = lds_w + (uint32_t)slot_of(j) * (2 * C::TILE_BYTES) + C::TILE_BYTES;
#pragma unroll
            for (int d = 0; d < C::DMA; d++) {
                const uint64_t row = *reinterpret_cast<const uint64_t*>(reinterpret_cast<const char*>(vrow_at) +
                                                                        (src[d] & 0xffffu));
                dma_gather16_nt(row + (src[d] >> 16), lds + 1024 * d);
            }
        };

        // The first tiles leave before the Q loads; the wait for Q drains them, once.
        if (my_tiles > 0) {
#pragma unroll
            for (int j = 0; j < C::SLOTS; j++) {
                issue_tab(j);
            }
            __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
#pragma unroll
            for (int j = 0; j < C::SLOTS; j++) {
                if (j < my_tiles) {
                    issue_k(j);
                    issue_v(j);
                }
            }
        }
        V8 qreg[C::NS];
        {
            const char* qrow = p.q + (int64_t)(seq.q0 + tok) * p.q_st + head * p.q_sh + 16 * g;
#pragma unroll
            for (int s = 0; s < C::NS; s++) {
                qreg[s] = *reinterpret_cast<const V8*>(qrow + 32 * s);
            }
#pragma unroll
            for (int s = 0; s < C::NS; s++) {
                qreg[s] = col_valid ? (p.q_sign < 0.0f ? -qreg[s] : qreg[s]) : V8{};
            }
        }
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));

        f16x oacc[C::NDT];
#pragma unroll
        for (int dt = 0; dt < C::NDT; dt++) {
            oacc[dt] = f16x{};
        }
        float m_run = -INFINITY, l_run = 0.0f;

        ValueScale vscale;

        for (int j = 0; j < my_tiles; j++) {
            const int kt0 = tile_key(j);
            const bool more = j + C::SLOTS < my_tiles; // a tile is issued into this one's slot
            const bool next = C::SLOTS > 1 && j + 1 < my_tiles; // the other slot is in flight
            // K(j) landed (and the entries of tile j + SLOTS): V(j) is younger, and the
            // other slot's tiles
            if (next) {
                __builtin_amdgcn_s_waitcnt(waitcnt_vm(C::V_COPIES + (C::SLOTS - 1) * (C::K_COPIES + C::V_COPIES)));
            } else {
                __builtin_amdgcn_s_waitcnt(waitcnt_vm(C::V_COPIES));
            }
            const char* const sk = wsm + slot_of(j) * (2 * C::TILE_BYTES);
            const char* const sv = sk + C::TILE_BYTES;

            // S^T[key][col] = K Q^T
            f16x sacc[1] = {f16x{}};
            f4 vs[I8 ? 4 : 1]; // the values' scales, of the keys of this lane's scores
            {
                const char* krow = sk + l32 * C::RB;
#pragma unroll
                for (int s = 0; s < C::NS; s++) {
                    V8 a;
                    if constexpr (I8) {
                        a = widen_int8<T>(*reinterpret_cast<const i2v*>(krow + ((s ^ swz8<D>(l32)) << 4) + 8 * g));
                    } else {
                        a = *reinterpret_cast<const V8*>(krow + (((2 * s + g) ^ paged_swz<D>(l32)) << 4));
                    }
                    sacc[0] = paged_mfma<T>(a, qreg[s], sacc[0]);
                }
                if constexpr (I8) {
                    const f4* sc = reinterpret_cast<const f4*>(aux + C::TAB_BYTES + 256 * slot_of(j)) + g;
                    f4 ks[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        ks[i] = sc[2 * i];
                        vs[i] = sc[8 + 2 * i];
                    }
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        sacc[0][e] *= ks[e >> 2][e & 3];
                    }
                }
            }
            if (more) {
                __builtin_amdgcn_s_waitcnt(waitcnt_lgkm(0)); // every read of K(j) has returned
                issue_k(j + C::SLOTS);
            }
            {
                const int a = row_lo - kt0 - 4 * g;
                const int bnd = row_hi - kt0 - 4 * g;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int off = 8 * (e >> 2) + (e & 3);
                    sacc[0][e] = (off < a || off > bnd) ? -INFINITY : sacc[0][e];
                }
            }
            if (p.tree != nullptr && kt0 + kTile > prefix) {
                tree_mask_scores<1>(sacc, tree_row, tree_n, prefix, kt0 + 4 * g);
            }
            float mx = max_tree<16>([&](int e) { return sacc[0][e]; });
            mx = pair_max(mx);
            const float m_new = fmaxf(m_run, mx * p.scale_log2e);
            const bool grow = m_new > m_run + kRescale;
            if (wave_any(grow)) {
                const float alpha = grow ? fast_exp2(m_run - m_new) : 1.0f;
                if (grow) {
                    m_run = m_new;
                }
                l_run *= alpha;
#pragma unroll
                for (int dt = 0; dt < C::NDT; dt++) {
                    oacc[dt] *= alpha;
                }
            }
            const float m_use = (m_run == -INFINITY) ? 0.0f : m_run;
            float pv[16];
            float ps[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < 16; e++) {
                pv[e] = fast_exp2(fmaf(sacc[0][e], p.scale_log2e, -m_use));
                ps[e & 3] += pv[e];
            }
            l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
            if constexpr (I8) {
                vscale.weigh<4>(pv, vs, oacc);
            }
            P8 pb[2];
#pragma unroll
            for (int e = 0; e < 16; e++) {
                pb[e >> 3][e & 7] = (P)pv[e];
            }

            // V(j) landed: the other slot's tiles are younger, and what was issued above
            if (more) {
                __builtin_amdgcn_s_waitcnt(
                    waitcnt_vm(C::K_COPIES + (C::SLOTS - 1) * (C::K_COPIES + C::V_COPIES)));
            } else if (next) {
                __builtin_amdgcn_s_waitcnt(waitcnt_vm((C::SLOTS - 1) * (C::K_COPIES + C::V_COPIES)));
            } else {
                __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
            }
            // O^T += V^T P^T; V^T operand through transpose reads
            const int j16 = lane & 15;
#pragma unroll
            for (int u = 0; u < 2; u++) {
#pragma unroll
                for (int dt = 0; dt < C::NDT; dt++) {
                    P8 a;
                    if constexpr (I8) {
                        const int r = 16 * u + 8 * (j16 >> 3) + 4 * g + ((j16 >> 1) & 3);
                        const int c = 2 * dt + ((lane >> 4) & 1);
                        a = widen_int8<P>(read_tr8(sv + r * C::RB + ((c ^ swz8<D>(r)) << 4) + 8 * (j16 & 1)));
                    } else {
                        h4 half4[2];
#pragma unroll
                        for (int hh = 0; hh < 2; hh++) {
                            const int r = 16 * u + 8 * hh + 4 * g + (j16 >> 2);
                            const int d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (j16 & 3);
                            const char* addr = sv + r * C::RB + (((d >> 3) ^ paged_swz<D>(r)) << 4) + ((d & 7) << 1);
                            half4[hh] = lds_read_tr16(reinterpret_cast<const _Float16*>(addr));
                        }
                        a = __builtin_bit_cast(P8, __builtin_shufflevector(half4[0], half4[1], 0, 1, 2, 3, 4, 5, 6, 7));
                    }
                    oacc[dt] = paged_mfma<P>(a, pb[u], oacc[dt]);
                }
            }
            if (more) {
                __builtin_amdgcn_s_waitcnt(waitcnt_lgkm(0)); // every read of V(j) has returned
                issue_v(j + C::SLOTS);
            }
        }
        __builtin_amdgcn_s_waitcnt(0);

        // ---- merge of the waves (see finish_rows) and the rows out
        {
            constexpr int LDM = D + 4;
            constexpr int MERGE = C::WAVES / 2;
            float* const sm_o = reinterpret_cast<float*>(dsm);
            float* const sm_ml = sm_o + MERGE * 32 * LDM;
            __syncthreads();
            const float l_tot = pair_sum(l_run);
            if (g == 0) {
                *reinterpret_cast<float2*>(&sm_ml[(wave * 32 + l32) * 2]) = float2{m_run, l_tot};
            }
            __syncthreads();
            float mref = -INFINITY, lsum = 0.0f;
#pragma unroll
            for (int w = 0; w < C::WAVES; w++) {
                mref = fmaxf(mref, sm_ml[(w * 32 + l32) * 2]);
            }
#pragma unroll
            for (int w = 0; w < C::WAVES; w++) {
                lsum += sm_ml[(w * 32 + l32) * 2 + 1] * part_weight(sm_ml[(w * 32 + l32) * 2], mref);
            }
            float scale_w = part_weight(m_run, mref);
            if constexpr (I8) {
                scale_w *= vscale.factor();
            }
            if (whole) {
                scale_w *= lsum > 0.0f ? 1.0f / lsum : 0.0f;
            }
            float* const my_o = &sm_o[((wave % MERGE) * 32 + l32) * LDM + 4 * g];
            auto put_o = [&]() {
                if (col_valid) {
#pragma unroll
                    for (int dt = 0; dt < C::NDT; dt++) {
#pragma unroll
                        for (int e4 = 0; e4 < 4; e4++) {
                            *reinterpret_cast<f4*>(my_o + 32 * dt + 8 * e4) =
                                f4{oacc[dt][4 * e4], oacc[dt][4 * e4 + 1], oacc[dt][4 * e4 + 2], oacc[dt][4 * e4 + 3]};
                        }
                    }
                }
            };
#pragma unroll
            for (int dt = 0; dt < C::NDT; dt++) {
                oacc[dt] *= scale_w;
            }
            if (wave >= MERGE) {
                put_o();
            }
            __syncthreads();
            if (wave < MERGE && col_valid) {
#pragma unroll
                for (int dt = 0; dt < C::NDT; dt++) {
#pragma unroll
                    for (int e4 = 0; e4 < 4; e4++) {
                        const f4 x = *reinterpret_cast<const f4*>(my_o + 32 * dt + 8 * e4);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            oacc[dt][4 * e4 + e] += x[e];
                        }
                    }
                }
            }
            if (wave < MERGE) {
                put_o(); // its own slot, read above by the same lanes
            }
            const int64_t slot = walk.slot();
            float* const part_o = p.part_o + slot * (kRows * D);
            if (!whole && tid < n_rows) { // threads 0 .. 31 hold mref, lsum of column tid
                *reinterpret_cast<float2*>(p.part_ml + (slot * kRows + tid) * 2) = float2{mref, lsum};
            }
            if (!whole && walk.at == 0) {
                rec = PagedRecord{n_rows, seq.q0, r0, h, walk.last_wg(), {}};
            }
            __syncthreads();
            for (int e = tid; e < n_rows * (D / 4); e += C::THREADS) {
                const int col = e / (D / 4);
                const int d = 4 * (e - col * (D / 4));
                f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < MERGE; w++) {
                    acc += *reinterpret_cast<const f4*>(&sm_o[(w * 32 + col) * LDM + d]);
                }
                if (whole) {
                    const int tk = (r0 + col) / G;
                    *reinterpret_cast<V4*>(p.o + (int64_t)(seq.q0 + tk) * p.o_st + (h * G + r0 + col - tk * G) * p.o_sh +
                                           2 * d) = __builtin_convertvector(acc, V4);
                } else {
                    *reinterpret_cast<f4*>(&part_o[col * D + d]) = acc;
                }
            }
            __syncthreads(); // the next item's copies overwrite the merge area
        }
        walk.next();
    }
    if (tid == 0) {
        p.records[walk.wg] = rec;
    }
}

} // namespace

// Smallest share: a tile for every wave of a workgroup.
int paged_stream_attention(const PagedAttnArgs& a, PagedAttnParams& p, const PagedLaunch& l, hipStream_t stream,
                           std::string& err) {
    return paged_for_type(a, [&](auto t, auto d, auto i8) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        constexpr bool I8 = decltype(i8)::value;
        using C = StreamCfg<D, I8>;
        return paged_launch<kRows, kTile>(a, reinterpret_cast<const void*>(&paged_stream<T, D, I8>), C::THREADS,
                                          C::WAVES, p, l, stream, err, [&](dim3 grid) {
                                              hipLaunchKernelGGL((paged_stream<T, D, I8>), grid, dim3(C::THREADS), 0,
                                                                 stream, p);
                                          });
    });
}

} // namespace rdna_amd
