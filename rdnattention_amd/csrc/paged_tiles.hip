// Paged attention of many rows per sequence and kv head (prompts, chunks of
// them, trees of drafts): out = softmax(c Q K^T) V over the pages of each
// sequence.
//
// Bound by the matrix cores where the rows fill the tiles.  A workgroup's waves
// hold 32 rows each of one kv head's rows (token after token, the G heads of a
// token side by side, so a chunk of few tokens fills the tiles too) and share
// 64-key tiles of K and V in LDS, two slots deep: the next tile's copies are
// issued as the present one is begun, one barrier per tile.  A row of a tile is
// found through the page table as in paged_stream.hip, the work dealt in equal
// shares of key tiles (PagedWalk), which also splits the keys of a call of few
// row tiles over the chip.
#include "paged_launch.hpp"

namespace rdna_amd {
namespace {

constexpr int kBN = 64;
constexpr float kRescale = 8.0f;

template <int D, bool I8>
struct TileCfg {
    // eight waves; above D = 128 four, one per SIMD, whose O takes up to 128 registers
    static constexpr int WAVES = D <= 128 ? 8 : 4;
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int WAVES_PER_SIMD = D <= 32 ? 4 : (D <= 128 ? 2 : 1);
    static constexpr int ROWS = 32 * WAVES;
    static constexpr int RB = 2 * D;
    static constexpr int KCH = D / 8;
    static constexpr int TILE_BYTES = kBN * RB;
    // the waves' table entries; of int8 the scales of two slots' keys and values
    static constexpr int TAB_BYTES = I8 ? 2 * 2 * kBN * 4 : WAVES * 256;
    static constexpr int NS = D / 16;
    static constexpr int NDT = D / 32;
    static constexpr int DMA = TILE_BYTES / 1024;                  // 1 KB copies of a tile
    static constexpr int PER = (DMA + WAVES - 1) / WAVES;          // of a wave
    static constexpr int CHUNKS = kBN * D / 16;                    // 16-byte chunks of an int8 tile
    static constexpr int NCH = (CHUNKS + THREADS - 1) / THREADS;   // per thread
    static_assert(4 * TILE_BYTES + TAB_BYTES <= 160 * 1024, "tiles fit the LDS");
};

template <class T, int D, bool I8>
__global__ __launch_bounds__((TileCfg<D, I8>::THREADS), (TileCfg<D, I8>::WAVES_PER_SIMD)) void paged_tiles(
    PagedAttnParams p) {
    using C = TileCfg<D, I8>;
    using V8 = typename PagedVec<T>::v8;
    using V4 = typename PagedVec<T>::v4;
    using P = std::conditional_t<I8, _Float16, T>; // weights and values, see paged_stream
    using P8 = typename PagedVec<P>::v8;
    // K and V of slot 0, of slot 1; the waves' table entries
    __shared__ __attribute__((aligned(16))) char dsm[4 * C::TILE_BYTES + C::TAB_BYTES];

    const int tid = threadIdx.x;
    const int wave = uniform(tid >> 6);
    const int lane = tid & 63;
    const int l32 = lane & 31;
    const int g = lane >> 5;
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(dsm);
    const uint32_t* const tab = reinterpret_cast<const uint32_t*>(dsm + 4 * C::TILE_BYTES) + 64 * wave;
    const uint32_t lds_tab = lds0 + 4 * C::TILE_BYTES + 256 * wave;
    const uint32_t page_mask = (1u << p.c.lps) - 1u;

    if (p.zero_tail != 0) {
        zero_tail_rows<D>(p);
    }
    PagedRecord rec = {};
    // row tiles of one head, which read the same keys, through one L2
    PagedWalk<C::ROWS, kBN> walk(p.work, by_xcd(blockIdx.x, p.work.n_wg));

    while (walk.more()) {
        const PagedSeq seq = walk.seq;
        const PagedTile item = walk.tile;
        const bool whole = walk.whole();
        const int h = walk.h;
        const int G = p.work.G;
        const int r0 = walk.rt * C::ROWS;
        const int n_rows = min(C::ROWS, seq.n * G - r0);
        const int wr0 = 32 * wave; // of the item
        const int col = wr0 + l32;
        const bool col_valid = col < n_rows;
        const bool active = wr0 < n_rows; // the wave
        const int tok = col_valid ? (r0 + col) / G : r0 / G;
        const int head = h * G + (col_valid ? r0 + col - tok * G : 0);
        const MaskSpec mask = paged_mask(p.work.mask, seq);
        int row_lo, row_hi;
        row_key_bounds(mask, tok, row_lo, row_hi);
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
        // the wave's classes of key tiles (see TileClasses)
        const TileClasses cls =
            active ? tile_classes<kBN>(mask, uniform((r0 + wr0) / G), uniform((r0 + min(wr0 + 32, n_rows) - 1) / G))
                   : TileClasses{1, 0, 1, 0};
        const int tree_from = p.tree != nullptr ? prefix : INT32_MAX; // keys from here on are under the tree's mask

        const int t0 = item.first + walk.at;
        const int nt = item.hi >= item.lo ? walk.count() : 0;
        const char* const kbase = p.c.k + h * p.c.k_sh;
        const char* const vbase = p.c.v + h * p.c.v_sh;
        const int32_t* const table = p.c.table + walk.b * p.c.table_s;

        // ---- 16-bit pages: copy d of a tile writes its LDS bytes 1024 d + 16 lane;
        // wave w has copies w, w + WAVES, ...
        i32x4_t tab_rsrc = make_rsrc_v(table, (uint32_t)p.c.width * 4u);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            tab_rsrc[e] = uniform(tab_rsrc[e]);
        }
        auto issue_tab = [&](int i) {
            dma_load4(tab_rsrc, (uint32_t)(((t0 + i) * kBN + lane) >> p.c.lps) * 4u, lds_tab);
        };
        auto issue_tile = [&](int i) { // its entries have landed
            const uint32_t slot = lds0 + (uint32_t)(i & 1) * (2 * C::TILE_BYTES);
            uint64_t ka[C::PER], va[C::PER];
#pragma unroll
            for (int c = 0; c < C::PER; c++) {
                const int d = wave + C::WAVES * c;
                const int n = 64 * (d < C::DMA ? d : 0) + lane;
                const int r = n / C::KCH;
                const uint32_t chunk = (uint32_t)((n - r * C::KCH) ^ paged_swz<D>(r)) * 16u;
                const int key = (t0 + i) * kBN + r;
                const bool seen = key >= item.lo && key <= item.hi;
                const uint32_t pg = tab[r];
                const uint64_t pe = pg < (uint32_t)p.c.pages ? pg : 0u;
                const uint64_t off = (uint32_t)key & page_mask;
                const uint64_t zero = reinterpret_cast<uint64_t>(kPagedZeroRow);
                ka[c] = (seen ? reinterpret_cast<uint64_t>(kbase) + pe * (uint64_t)p.c.k_sp + off * (uint64_t)p.c.k_st
                              : zero) + chunk;
                va[c] = (seen ? reinterpret_cast<uint64_t>(vbase) + pe * (uint64_t)p.c.v_sp + off * (uint64_t)p.c.v_st
                              : zero) + chunk;
            }
            __builtin_amdgcn_s_waitcnt(waitcnt_lgkm(0)); // the entries are read
#pragma unroll
            for (int c = 0; c < C::PER; c++) {
                const int d = wave + C::WAVES * c;
                if (C::DMA % C::WAVES == 0 || d < C::DMA) {
                    dma_gather16(ka[c], slot + 1024 * d);
                    dma_gather16(va[c], slot + C::TILE_BYTES + 1024 * d);
                }
            }
        };

        // ---- int8 pages: through registers, widened exactly (once for all waves); the
        // scales beside them
        constexpr int RCH = D / 16;
        float* const scales = reinterpret_cast<float*>(dsm + 4 * C::TILE_BYTES); // [slot][keys, values][kBN]
        auto chunk_row = [&](int c) { return (C::THREADS * c + tid) / RCH % kBN; };
        int32_t ent[C::NCH];
        i4 kraw[C::NCH], vraw[C::NCH];
        float ksc[C::NCH], vsc[C::NCH];
        auto load_entries = [&](int i) {
#pragma unroll
            for (int c = 0; c < C::NCH; c++) {
                const int e = ((t0 + i) * kBN + chunk_row(c)) >> p.c.lps;
                ent[c] = table[min(e, p.c.width - 1)];
            }
        };
        auto load_raw = [&](int i) {
#pragma unroll
            for (int c = 0; c < C::NCH; c++) {
                const int key = (t0 + i) * kBN + chunk_row(c);
                const bool seen = key >= item.lo && key <= item.hi;
                const int64_t pg = (uint32_t)ent[c] < (uint32_t)p.c.pages ? ent[c] : 0;
                const int64_t off = (uint32_t)key & page_mask;
                const int ch = 16 * (tid % RCH);
                kraw[c] = *reinterpret_cast<const i4*>(kbase + pg * p.c.k_sp + off * p.c.k_st + ch);
                vraw[c] = *reinterpret_cast<const i4*>(vbase + pg * p.c.v_sp + off * p.c.v_st + ch);
                const float a = p.c.ks[pg * p.c.ks_sp + off * p.c.ks_st + h * p.c.ks_sh];
                const float b = p.c.vs[pg * p.c.vs_sp + off * p.c.vs_st + h * p.c.vs_sh];
                ksc[c] = seen ? a : 0.0f;
                vsc[c] = seen ? b : 0.0f;
            }
        };
        auto store_raw = [&](int i) {
            char* const sk = dsm + (i & 1) * (2 * C::TILE_BYTES);
#pragma unroll
            for (int c = 0; c < C::NCH; c++) {
                const int r = chunk_row(c);
                const int cl = 2 * (tid % RCH);
                if (C::CHUNKS % C::THREADS != 0 && C::THREADS * c + tid >= C::CHUNKS) {
                    continue;
                }
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    char* const at = sk + r * C::RB + (((cl + x) ^ paged_swz<D>(r)) << 4);
                    *reinterpret_cast<V8*>(at) = widen_int8<T>(i2v{kraw[c][2 * x], kraw[c][2 * x + 1]});
                    *reinterpret_cast<P8*>(at + C::TILE_BYTES) = widen_int8<P>(i2v{vraw[c][2 * x], vraw[c][2 * x + 1]});
                }
                if (cl == 0) {
                    scales[(i & 1) * 2 * kBN + r] = ksc[c];
                    scales[(i & 1) * 2 * kBN + kBN + r] = vsc[c];
                }
            }
        };

        if (nt > 0) {
            if constexpr (I8) {
                load_entries(0);
                load_raw(0);
                load_entries(1);
            } else {
                issue_tab(0);
                __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
                issue_tile(0);
                issue_tab(1);
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
        if constexpr (I8) {
            if (nt > 0) {
                store_raw(0);
                load_raw(1);
                load_entries(2);
            }
        }

        f16x oacc[C::NDT];
#pragma unroll
        for (int dt = 0; dt < C::NDT; dt++) {
            oacc[dt] = f16x{};
        }
        float m_run = -INFINITY, l_run = 0.0f;
        ValueScale vscale;

        for (int i = 0; i < nt; i++) {
            // this wave's copies of tile i (and the entries of i + 1) have landed; behind
            // the barrier every wave's, and no wave reads tile i - 1 any more
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if constexpr (!I8) {
                if (i + 1 < nt) {
                    issue_tile(i + 1);
                    issue_tab(i + 2);
                }
            }
            const char* const sk = dsm + (i & 1) * (2 * C::TILE_BYTES);
            const char* const sv = sk + C::TILE_BYTES;
            const int kt0 = (t0 + i) * kBN;
            const int what = tile_class(cls, t0 + i);
            if (what != 0) {
                f16x sacc[2] = {f16x{}, f16x{}};
#pragma unroll
                for (int s = 0; s < C::NS; s++) {
#pragma unroll
                    for (int kt = 0; kt < 2; kt++) {
                        const int r = 32 * kt + l32;
                        const V8 a =
                            *reinterpret_cast<const V8*>(sk + r * C::RB + (((2 * s + g) ^ paged_swz<D>(r)) << 4));
                        sacc[kt] = paged_mfma<T>(a, qreg[s], sacc[kt]);
                    }
                }
                if constexpr (I8) {
                    const f4* sc = reinterpret_cast<const f4*>(scales + (i & 1) * 2 * kBN) + g;
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        const f4 ks = sc[2 * x];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            sacc[x >> 2][4 * (x & 3) + e] *= ks[e];
                        }
                    }
                }
                if (what == 2) {
                    const int a = row_lo - kt0 - 4 * g;
                    const int bnd = row_hi - kt0 - 4 * g;
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        const int off = 32 * (e >> 4) + 8 * ((e & 15) >> 2) + (e & 3);
                        sacc[e >> 4][e & 15] = (off < a || off > bnd) ? -INFINITY : sacc[e >> 4][e & 15];
                    }
                }
                if (kt0 + kBN > tree_from) {
                    tree_mask_scores<2>(sacc, tree_row, tree_n, prefix, kt0 + 4 * g);
                }
                float mx = max_tree<32>([&](int e) { return sacc[e >> 4][e & 15]; });
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
                float pv[32];
                float ps[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    pv[e] = fast_exp2(fmaf(sacc[e >> 4][e & 15], p.scale_log2e, -m_use));
                    ps[e & 3] += pv[e];
                }
                l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
                if constexpr (I8) {
                    const f4* sc = reinterpret_cast<const f4*>(scales + (i & 1) * 2 * kBN + kBN) + g;
                    f4 vs[8];
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        vs[x] = sc[2 * x];
                    }
                    vscale.weigh<8>(pv, vs, oacc);
                }
                P8 pb[4];
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    pb[e >> 3][e & 7] = (P)pv[e];
                }
                const int j16 = lane & 15;
#pragma unroll
                for (int u = 0; u < 4; u++) {
#pragma unroll
                    for (int dt = 0; dt < C::NDT; dt++) {
                        h4 half4[2];
#pragma unroll
                        for (int hh = 0; hh < 2; hh++) {
                            const int r = 16 * u + 8 * hh + 4 * g + (j16 >> 2);
                            const int d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (j16 & 3);
                            const char* addr =
                                sv + r * C::RB + (((d >> 3) ^ paged_swz<D>(r)) << 4) + ((d & 7) << 1);
                            half4[hh] = lds_read_tr16(reinterpret_cast<const _Float16*>(addr));
                        }
                        const h8 a = __builtin_shufflevector(half4[0], half4[1], 0, 1, 2, 3, 4, 5, 6, 7);
                        oacc[dt] = paged_mfma<P>(__builtin_bit_cast(P8, a), pb[u], oacc[dt]);
                    }
                }
            }
            if constexpr (I8) {
                if (i + 1 < nt) {
                    store_raw(i + 1); // its slot was last read before this tile's barrier
                    load_raw(i + 2);
                    load_entries(i + 3);
                }
            }
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads(); // the next item's copies overwrite the slots

        const float l_tot = pair_sum(l_run);
        const float unit = I8 ? vscale.factor() : 1.0f; // of O
        if (whole) {
            const float inv = l_tot > 0.0f ? unit / l_tot : 0.0f;
            if (col_valid) {
                char* const orow = p.o + (int64_t)(seq.q0 + tok) * p.o_st + head * p.o_sh;
#pragma unroll
                for (int dt = 0; dt < C::NDT; dt++) {
#pragma unroll
                    for (int qq = 0; qq < 4; qq++) {
                        const f4 x = f4{oacc[dt][4 * qq], oacc[dt][4 * qq + 1], oacc[dt][4 * qq + 2],
                                        oacc[dt][4 * qq + 3]} * inv;
                        *reinterpret_cast<V4*>(orow + 2 * (32 * dt + 8 * qq + 4 * g)) = __builtin_convertvector(x, V4);
                    }
                }
            }
        } else {
            const int64_t slot = walk.slot();
            if (col_valid) {
                store_partial<C::NDT>(oacc, m_run, l_tot, g == 0, p.part_o, p.part_ml, slot * p.slot_rows + col, D, 0, g,
                                      [&](int) { return f4{unit, unit, unit, unit}; });
            }
            if (walk.at == 0) {
                rec = PagedRecord{n_rows, seq.q0, r0, h, walk.last_wg(), {}};
            }
        }
        walk.next();
    }
    if (tid == 0) {
        p.records[walk.wg] = rec;
    }
}

} // namespace

// Smallest share: four key tiles.
int paged_tile_attention(const PagedAttnArgs& a, PagedAttnParams& p, const PagedLaunch& l, hipStream_t stream,
                         std::string& err) {
    return paged_for_type(a, [&](auto t, auto d, auto i8) {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        constexpr bool I8 = decltype(i8)::value;
        using C = TileCfg<D, I8>;
        return paged_launch<C::ROWS, kBN>(a, reinterpret_cast<const void*>(&paged_tiles<T, D, I8>), C::THREADS, 1, 4, p, l,
                                          stream, err, [&](dim3 grid) {
                                              hipLaunchKernelGGL((paged_tiles<T, D, I8>), grid, dim3(C::THREADS), 0,
                                                                 stream, p);
                                          });
    });
}

} // namespace rdna_amd
