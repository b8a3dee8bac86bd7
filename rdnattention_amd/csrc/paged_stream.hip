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
#include "paged_attn.hpp"

#include "paged_launch.hpp"

namespace rdna_amd {
namespace {

constexpr int kRows = 32; // rows per item: columns of the MFMAs
constexpr int kTile = 32; // keys per wave tile
constexpr int kManyHeads = 512; // kv heads of all sequences: two per CU
constexpr float kRescale = 8.0f;
constexpr int kDepth = 4; // MFMA operands in flight

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

// 16-byte chunk swizzle of row r of an int8 tile: rows of 64 or 128 bytes, the 64
// banks 256, so rows r and r + 4 or r + 2 start in the same bank
template <int D>
__device__ __forceinline__ int swz8(int r) {
    return D == 64 ? (r >> 2) & 3 : (r >> 1) & 7;
}

template <class T, int D, bool I8, int WV>
__global__ __launch_bounds__((StreamCfg<D, I8, WV>::THREADS), (StreamCfg<D, I8, WV>::WAVES_PER_SIMD)) void paged_stream(
    PagedAttnParams p) {
    using C = StreamCfg<D, I8, WV>;
    using V8 = typename PagedVec<T>::v8;
    using V4 = typename PagedVec<T>::v4;
    // weights and values meet in P: int8 values are exact in fp16, whose weights
    // round finer than bf16's
    using P = std::conditional_t<I8, _Float16, T>;
    using P8 = typename PagedVec<P>::v8;
    __shared__ __attribute__((aligned(16))) char dsm[C::LDS_BYTES];

    const int tid = threadIdx.x;
    const int wave = uniform(tid >> 6);
    const int lane = tid & 63;
    const int l32 = lane & 31;
    const int g = lane >> 5;
    // K tile, V tile; then table entries, scales, row addresses
    char* const wsm = dsm + wave * C::WAVE_BYTES;
    char* const aux = wsm + 2 * C::TILE_BYTES;
    const uint32_t lds_w = (uint32_t)reinterpret_cast<uintptr_t>(wsm);
    const uint32_t lds_aux = lds_w + 2 * C::TILE_BYTES;
    uint64_t* const rows_at = reinterpret_cast<uint64_t*>(aux + C::TAB_BYTES + C::SCALE_BYTES); // K rows, V rows

    if (p.zero_tail != 0) {
        zero_tail_rows<D>(p);
    }
    PagedRecord rec = {};
    // Heads of int8 pages next to each other on one XCD: a line of scales holds those
    // of many heads.  16-bit pages share no lines, and spread over the XCDs they are
    // read faster.  (us, neighbours on one XCD / spread: int8 32 x 8192 keys of 8 heads
    // 117 / 124, 32 ragged ones 143 / 154; fp16 16 x 18432 of 8 heads, D = 128 204 / 197,
    // D = 64 124 / 118, 8 x 16384 of 16 heads 182 / 173, ragged 193 / 193.)
    PagedWalk<kRows, kTile, false, 0> walk(p.work, I8 ? by_xcd(blockIdx.x, p.work.n_wg) : (int32_t)blockIdx.x);

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
        const int h = uniform(walk.h);
        const int G = p.work.G;
        const int r0 = uniform(walk.rt) * kRows;
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

        const int t0 = uniform(item.first + walk.begin());
        const int nt = uniform(item.hi >= item.lo ? walk.count() : 0);
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
        // Table entries come in batches of 64, those of the wave's next 64 / n tiles, n
        // = max(1, 32 / page size) entries each: a copy per tile would be one more
        // beside the tile's own sixteen, and cost as much to issue as any.  (16 bf16
        // sequences of 4000 to 32768 keys, D = 128: 190.4 us with a copy per tile.)
        const int log_n = max(0, 5 - p.c.lps);
        const int log_b = 6 - log_n; // tiles of a batch
        auto issue_tab = [&](int batch) {
            const int t = (batch << log_b) + (lane >> log_n);
            const int key = tile_key(t) + ((lane & ((1 << log_n) - 1)) << p.c.lps);
            dma_load4(tab_rsrc, (uint32_t)(key >> p.c.lps) * 4u, (uint32_t)uniform((int)lds_aux + 256 * (batch & 1)));
        };
        // The row addresses of tile j, from its entries: lanes 0 - 31 leave K row l32's,
        // the others V row l32's.  One tile ahead, before the S of another is computed,
        // so that the copies leave as soon as their slot is free.
        uint64_t scale_at = 0;
        auto find_rows = [&](int j) {
            const int key = tile_key(j) + l32;
            const uint32_t pg =
                reinterpret_cast<const uint32_t*>(aux)[64 * ((j >> log_b) & 1) + ((j & ((1 << log_b) - 1)) << log_n) +
                                                       (l32 >> p.c.lps)];
            const bool seen = key >= item.lo && key <= item.hi;
            const uint64_t pe = pg < (uint32_t)p.c.pages ? pg : 0u;
            const uint64_t off = (uint32_t)key & page_mask;
            const uint64_t zero = reinterpret_cast<uint64_t>(kPagedZeroRow);
            const uint64_t base = reinterpret_cast<uint64_t>(g == 0 ? kbase : vbase);
            const uint64_t sp = g == 0 ? p.c.k_sp : p.c.v_sp, st = g == 0 ? p.c.k_st : p.c.v_st;
            rows_at[lane] = seen ? base + pe * sp + off * st : zero;
            if constexpr (I8) {
                const uint64_t sb = reinterpret_cast<uint64_t>(g == 0 ? p.c.ks : p.c.vs);
                const uint64_t ssp = g == 0 ? p.c.ks_sp : p.c.vs_sp, sst = g == 0 ? p.c.ks_st : p.c.vs_st;
                const uint64_t ssh = g == 0 ? p.c.ks_sh : p.c.vs_sh;
                scale_at = seen ? sb + 4 * (pe * ssp + off * sst + h * ssh) : zero;
            }
        };
        uint64_t from[C::DMA]; // of each copy, this lane's 16 bytes
        auto read_rows = [&](int values) {
#pragma unroll
            for (int d = 0; d < C::DMA; d++) {
                from[d] = *reinterpret_cast<const uint64_t*>(reinterpret_cast<const char*>(rows_at + kTile * values) +
                                                             (src[d] & 0xffffu)) +
                          (src[d] >> 16);
            }
        };
        // K tile j and its scales
        auto issue_k = [&]() {
#pragma unroll
            for (int d = 0; d < C::DMA; d++) {
                dma_gather16_nt(from[d], lds_w + 1024 * d);
            }
            if constexpr (I8) { // the keys' scales from lanes 0 - 31, the values'
                dma_gather4(scale_at, lds_aux + C::TAB_BYTES);
            }
        };
        auto issue_v = [&]() {
#pragma unroll
            for (int d = 0; d < C::DMA; d++) {
                dma_gather16_nt(from[d], lds_w + C::TILE_BYTES + 1024 * d);
            }
        };

        // The first tiles leave before the Q loads; the wait for Q drains them, once.
        if (my_tiles > 0) {
            issue_tab(0);
            issue_tab(1);
            __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
            find_rows(0);
            read_rows(0);
            issue_k();
            read_rows(1);
            issue_v();
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
            const bool more = j + 1 < my_tiles;
            // K(j) landed: only V(j) is younger
            __builtin_amdgcn_s_waitcnt(waitcnt_vm(C::V_COPIES));
            const char* const sk = wsm;
            const char* const sv = sk + C::TILE_BYTES;
            if (more) {
                find_rows(j + 1);
            }

            // S^T[key][col] = K Q^T
            f16x sacc[1] = {f16x{}};
            f4 vs[I8 ? 4 : 1]; // the values' scales, of the keys of this lane's scores
            {
                const char* krow = sk + l32 * C::RB;
                using Raw = std::conditional_t<I8, i2v, V8>;
                operand_stream<C::NS, kDepth>(
                    [&](int s) {
                        return *reinterpret_cast<const Raw*>(
                            krow + (I8 ? ((s ^ swz8<D>(l32)) << 4) + 8 * g : ((2 * s + g) ^ paged_swz<D>(l32)) << 4));
                    },
                    [&](int s, Raw a) {
                        if constexpr (I8) {
                            sacc[0] = paged_mfma<T>(widen_int8<T>(a), qreg[s], sacc[0]);
                        } else {
                            sacc[0] = paged_mfma<T>(a, qreg[s], sacc[0]);
                        }
                    });
                if constexpr (I8) {
                    const f4* sc = reinterpret_cast<const f4*>(aux + C::TAB_BYTES) + g;
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
            // Once the first tile of a batch has its addresses, the batch before it is
            // done with, and the one after it is copied there, before K(j + 1), which is
            // awaited for tile j + 1: earlier than these entries are wanted (a batch has
            // two tiles at least).
            const bool entries = more && ((j + 1) & ((1 << log_b) - 1)) == 0;
            if (more) {
                read_rows(0);
                __builtin_amdgcn_s_waitcnt(waitcnt_lgkm(0)); // every read of K(j) has returned
                if (entries) {
                    issue_tab(((j + 1) >> log_b) + 1);
                }
                issue_k();
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

            // V(j) landed: only what was issued above is younger
            if (entries) {
                __builtin_amdgcn_s_waitcnt(waitcnt_vm(C::K_COPIES + 1));
            } else if (more) {
                __builtin_amdgcn_s_waitcnt(waitcnt_vm(C::K_COPIES));
            } else {
                __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
            }
            // O^T += V^T P^T; V^T operand through transpose reads
            const int j16 = lane & 15;
            using VRaw = std::conditional_t<I8, i2v, h8>;
            operand_stream<2 * C::NDT, kDepth>(
                [&](int i) {
                    const int u = i / C::NDT, dt = i % C::NDT;
                    if constexpr (I8) {
                        const int r = 16 * u + 8 * (j16 >> 3) + 4 * g + ((j16 >> 1) & 3);
                        const int c = 2 * dt + ((lane >> 4) & 1);
                        return read_tr8(sv + r * C::RB + ((c ^ swz8<D>(r)) << 4) + 8 * (j16 & 1));
                    } else {
                        h4 half4[2];
#pragma unroll
                        for (int hh = 0; hh < 2; hh++) {
                            const int r = 16 * u + 8 * hh + 4 * g + (j16 >> 2);
                            const int d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (j16 & 3);
                            const char* addr = sv + r * C::RB + (((d >> 3) ^ paged_swz<D>(r)) << 4) + ((d & 7) << 1);
                            half4[hh] = lds_read_tr16(reinterpret_cast<const _Float16*>(addr));
                        }
                        return h8(__builtin_shufflevector(half4[0], half4[1], 0, 1, 2, 3, 4, 5, 6, 7));
                    }
                },
                [&](int i, VRaw a) {
                    const int u = i / C::NDT, dt = i % C::NDT;
                    if constexpr (I8) {
                        oacc[dt] = paged_mfma<P>(widen_int8<P>(a), pb[u], oacc[dt]);
                    } else {
                        oacc[dt] = paged_mfma<P>(__builtin_bit_cast(P8, a), pb[u], oacc[dt]);
                    }
                });
            if (more) {
                read_rows(1);
                __builtin_amdgcn_s_waitcnt(waitcnt_lgkm(0)); // every read of V(j) has returned
                issue_v();
            }
        }
        __builtin_amdgcn_s_waitcnt(0);

        // ---- merge of the waves through LDS, each wave's rows once, and the rows out
        {
            constexpr int LDM = D + 4;
            float* const sm_o = reinterpret_cast<float*>(dsm);
            float* const sm_ml = sm_o + C::WAVES * kRows * LDM;
            const float l_tot = pair_sum(l_run);
            __syncthreads(); // the waves are done with their tiles
            if (g == 0) {
                *reinterpret_cast<float2*>(&sm_ml[(wave * 32 + l32) * 2]) = float2{m_run, l_tot};
            }
            if (col_valid) {
                const float unit = I8 ? vscale.factor() : 1.0f; // of O
                float* const my_o = &sm_o[(wave * n_rows + l32) * LDM + 4 * g];
#pragma unroll
                for (int dt = 0; dt < C::NDT; dt++) {
#pragma unroll
                    for (int e4 = 0; e4 < 4; e4++) {
                        *reinterpret_cast<f4*>(my_o + 32 * dt + 8 * e4) =
                            f4{oacc[dt][4 * e4], oacc[dt][4 * e4 + 1], oacc[dt][4 * e4 + 2], oacc[dt][4 * e4 + 3]} *
                            unit;
                    }
                }
            }
            const int64_t slot = (int64_t)walk.slot() * p.slot_rows;
            if (!whole && walk.begin() == 0) {
                rec = PagedRecord{n_rows, seq.q0, r0, h, walk.last_wg(), {}};
            }
            __syncthreads();
            for (int e = tid; e < n_rows * (D / 4); e += C::THREADS) {
                const int col = e / (D / 4);
                const int d = 4 * (e - col * (D / 4));
                float2 ml[C::WAVES];
                float mref = -INFINITY, lsum = 0.0f;
#pragma unroll
                for (int w = 0; w < C::WAVES; w++) {
                    ml[w] = *reinterpret_cast<const float2*>(&sm_ml[(w * 32 + col) * 2]);
                    mref = fmaxf(mref, ml[w].x);
                }
                f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < C::WAVES; w++) {
                    const float wt = part_weight(ml[w].x, mref);
                    lsum += ml[w].y * wt;
                    // a wave that saw no key of this row adds nothing
                    const f4 x = *reinterpret_cast<const f4*>(&sm_o[(w * n_rows + col) * LDM + d]);
                    acc += ml[w].y != 0.0f ? x * wt : f4{0.0f, 0.0f, 0.0f, 0.0f};
                }
                if (whole) {
                    const int tk = (r0 + col) / G;
                    acc *= lsum > 0.0f ? 1.0f / lsum : 0.0f;
                    *reinterpret_cast<V4*>(p.o + (int64_t)(seq.q0 + tk) * p.o_st + (h * G + r0 + col - tk * G) * p.o_sh +
                                           2 * d) = __builtin_convertvector(acc, V4);
                } else {
                    *reinterpret_cast<f4*>(&p.part_o[(slot + col) * D + d]) = acc;
                    if (d == 0) {
                        *reinterpret_cast<float2*>(p.part_ml + (slot + col) * 2) = float2{mref, lsum};
                    }
                }
            }
            __syncthreads(); // the next item's copies overwrite the merge area
        }
        walk.next();
    }
    if (tid == 0) {
        p.records[walk.part.wg] = rec;
    }
}

} // namespace

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
