// The attention that each cached key has received from a call's rows, added to its
// weight: w_j = (decay w_j, or 0 where the key is one of the newest rows) + the sum over
// the rows i and the G heads of the key's kv head of exp(c q_i k_j - lse_i).
//
// The keys are the lanes of the matrix products (S = Q K^T, a row of Q to a register),
// so that a key's sum stays in its lane, whatever its page holds reaches no other key,
// and two workgroups that share a key leave their sums in order: no atomics, the same bits
// every time.
//   * few rows (up to 128 of a kv head): bound by HBM; K is read once for every 32 rows, by
//     those that see it
//   * more rows: bound by the exponentials beside the products.  A workgroup keeps a block of
//     keys in registers and its waves take the row tiles in turn, Q through LDS one tile
//     ahead
#include "fa_common.hpp"
#include "paged_attn.hpp"
#include "paged_launch.hpp"

#include <algorithm>

namespace rdna_amd {

float softmax_log2_scale(float scale);

namespace {

constexpr int kTile = 32;    // keys and rows of a product
// Up to this many rows x heads of a kv head by paged_weights_few, which goes over the keys for
// each 32 of them (launch_weights: fewer where waves of it are idle).  Sequences of 8192 keys, 8 kv
// heads, us by few / many for 32 rows, 64, 96, 128 (at 16 sequences K stays in the last-level
// cache, at 64, or 32 of D = 256, it does not):
//   16, bf16, D 64          28 / 98   53 / 103   76 / 108   99 / 113
//   16, bf16, D 128         48 / 154  91 / 166   132 / 181  174 / 192
//   16, the same, window 1024  28 / 136  52 / 142   78 / 146   103 / 151
//   16, int8, D 128         39 / 141  73 / 172   105 / 176  136 / 178
//   64, bf16, D 64          111       222 / 424  333 / 446  443 / 464
//   64, bf16, D 128         200       402 / 660  602 / 719  800 / 763
//   64, int8, D 128         130       255 / 674  379 / 668  506 / 690
//   32, bf16, D 256         175       345 / 764  519 / 834  693 / 929
constexpr int kFewMax = 128;
// one item per kv head of a sequence, its units blocks of keys
constexpr int kAllRows = 1 << 30;
constexpr float kLog2e = 1.4426950408889634f;

struct WeightsParams {
    PagedPages c;
    PagedWork work; // of few rows without a mask: every key has a weight
    PagedMask mask;
    const char* q;
    int64_t q_st, q_sh; // bytes
    const float* lse;
    int32_t Hq, Hkv;
    float scale_log2e; // |scale| log2(e)
    float q_sign;
    float decay;
    float* w;
    int64_t w_sp, w_st, w_sh;
    // blocks of keys that several workers share: sums by slot, as in PagedRecord, whose q0 is
    // the sequence and r0 the first key
    float* parts;
    PagedRecord* records;
};

// A row's log-sum-exp in log2 units, as what is subtracted in the exponent and a factor
// for the rest of the product lse log2(e), which 32 bits do not hold: the weights of a row
// would all be off by 2^-24 of the exponent.  A row that sees nothing has no weights.
struct RowLse {
    float sub, factor;
};
__device__ __forceinline__ RowLse row_lse(float lse) {
    const float hi = lse * kLog2e;
    float lo = fmaf(lse, kLog2e, -hi) + lse * 1.925963033500000e-08f; // log2(e) - kLog2e
    lo = fabsf(lo) < 1.0f ? lo : 0.0f;                                // infinities
    return lse == -INFINITY ? RowLse{INFINITY, 1.0f} : RowLse{hi, fast_exp2(-lo)};
}

// What a lane needs of key `key`, given its entry of the page table.
struct LaneKey {
    const char* k;
    float* w;      // null: no key, or no page
    float k_scale; // int8 pages
};

__device__ __forceinline__ int32_t key_entry(const WeightsParams& p, const PagedSeq& seq, const int32_t* table,
                                             int key) {
    return key < seq.len ? paged_page(p.c, table, key >> p.c.lps) : -1;
}

template <bool I8>
__device__ __forceinline__ LaneKey lane_key(const WeightsParams& p, int32_t entry, int h, int key) {
    LaneKey r;
    const int64_t page = entry >= 0 ? entry : 0;
    const int64_t off = key & ((1 << p.c.lps) - 1);
    r.k = entry >= 0 ? p.c.k + page * p.c.k_sp + off * p.c.k_st + h * p.c.k_sh
                     : reinterpret_cast<const char*>(kPagedZeroRow);
    r.w = entry >= 0 ? p.w + page * p.w_sp + off * p.w_st + h * p.w_sh : nullptr;
    r.k_scale = 1.0f;
    if constexpr (I8) {
        r.k_scale = entry >= 0 ? p.c.ks[page * p.c.ks_sp + off * p.c.ks_st + h * p.c.ks_sh] : 0.0f;
    }
    return r;
}

// A key's row in the MFMA layout: lane (l32, g) holds chunk x of row l32, a chunk being 16
// bytes of it.
template <int D, bool I8>
struct KeyRegs {
    static constexpr int N = I8 ? D / 32 : D / 16;
    i4 x[N];
    __device__ __forceinline__ void load(const char* row, int g) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            x[i] = *reinterpret_cast<const i4*>(row + 32 * i + 16 * g);
        }
    }
    // operand s of the product over D, which chunk_of_q(s) of the row of Q meets
    template <class T>
    __device__ __forceinline__ typename PagedVec<T>::v8 operand(int s) const {
        if constexpr (I8) {
            return widen_int8<T>(i2v{x[s >> 1][2 * (s & 1)], x[s >> 1][2 * (s & 1) + 1]});
        } else {
            return __builtin_bit_cast(typename PagedVec<T>::v8, x[s]);
        }
    }
};
template <bool I8>
__device__ __forceinline__ int chunk_of_q(int s, int g) {
    return I8 ? 4 * (s >> 1) + 2 * g + (s & 1) : 2 * s + g;
}

// Sum over the lane's 16 rows (base + 8 (e / 4) + 4 g + e % 4) of their weights on its key,
// times the rows' factors.  (Of many rows without: their errors of 2^-24 of an exponent are
// of either sign, and the registers hold another tile of keys.)
template <bool MASK, bool FACTOR>
__device__ __forceinline__ float sum_weights(const f16x& s, float c, const f4 (&sub)[4], const f4 (&factor)[4], int lo,
                                             int hi, float sum) {
    float part[4] = {sum, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 16; e++) {
        float p = fast_exp2(fmaf(s[e], c, -sub[e >> 2][e & 3]));
        if constexpr (MASK) {
            const int off = 8 * (e >> 2) + (e & 3);
            p = off < lo || off > hi ? 0.0f : p;
        }
        part[e & 3] = FACTOR ? fmaf(p, factor[e >> 2][e & 3], part[e & 3]) : part[e & 3] + p;
    }
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// The weight of a key from before the newest rows (is_old), or of one of theirs.
__device__ __forceinline__ float new_weight(const WeightsParams& p, bool is_old, float sum, float old) {
    return is_old && p.decay != 0.0f ? fmaf(p.decay, old, sum) : sum;
}

// Few rows.  The waves of a workgroup have the kv heads, eight at a time, of the same 32 keys
// (and of the next 32 where there are fewer heads), since the keys of a token lie side by
// side and a line of weights holds those of its heads.  Keys come by non-temporal HBM ->
// LDS copies, one tile ahead, each of whole rows, and so do the old weights, the scales
// of int8 and, 64 at a time, the page table's entries: no wait of the compiler's drains them.
// us for 16 bf16 sequences of 4000 to 32768 keys, 8 heads, D = 128: 107; with a workgroup's
// waves on one head 146 (30 of it for the weights' lines), keys loaded straight into the
// MFMA layout (32 bytes of each of 32 rows at a time) 133 to 137, one to three tiles ahead.
template <int D, bool I8>
struct FewCfg {
    static constexpr int WAVES = D <= 128 ? 8 : 4;
    static constexpr int RB = I8 ? D : 2 * D; // row bytes
    static constexpr int KCH = RB / 16;
    static constexpr int TILE_BYTES = kTile * RB;
    static constexpr int DMA = TILE_BYTES / 1024;
    // two tiles; two batches of 64 table entries; of both tiles 32 old weights and 32 scales;
    // row addresses; the rows' log-sum-exps
    static constexpr int TABS = 2 * TILE_BYTES, AUX = TABS + 2 * 256, ROWS = AUX + 2 * 256, LSE = ROWS + 256;
    static constexpr int WAVE_BYTES = LSE + 256;
    static_assert(WAVES * WAVE_BYTES <= 160 * 1024, "tiles fit the LDS");
};

template <class T, int D, bool I8>
__global__ __launch_bounds__((64 * FewCfg<D, I8>::WAVES)) void paged_weights_few(WeightsParams p) {
    using C = FewCfg<D, I8>;
    using V8 = typename PagedVec<T>::v8;
    constexpr int NS = D / 16, WAVES = C::WAVES;
    __shared__ __attribute__((aligned(16))) char dsm[WAVES * C::WAVE_BYTES];
    const int wave = uniform(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int l32 = lane & 31, g = lane >> 5;
    char* const wsm = dsm + wave * C::WAVE_BYTES;
    const uint32_t lds_w = (uint32_t)reinterpret_cast<uintptr_t>(wsm);
    uint64_t* const rows_at = reinterpret_cast<uint64_t*>(wsm + C::ROWS);
    float* const rows_lse = reinterpret_cast<float*>(wsm + C::LSE);
    const int side = min(p.Hkv, WAVES); // heads side by side,
    const int step = WAVES / side;      // and tiles
    const int slot = wave / side;
    const uint32_t page_mask = (1u << p.c.lps) - 1u;
    const uint64_t zero = reinterpret_cast<uint64_t>(kPagedZeroRow);
    // lane i of copy d writes bytes 1024 d + 16 i of a tile: stored chunk n % KCH of row n /
    // KCH, n = 64 d + i, which holds chunk (n % KCH) ^ swz(row)
    uint32_t src[C::DMA]; // row * 8 | chunk byte << 16
#pragma unroll
    for (int d = 0; d < C::DMA; d++) {
        const int n = 64 * d + lane;
        const int r = n / C::KCH;
        src[d] = (uint32_t)(r * 8) | (uint32_t)(((n - r * C::KCH) ^ (I8 ? swz8<D>(r) : paged_swz<D>(r))) * 16) << 16;
    }
    const int log_n = max(0, 5 - p.c.lps); // table entries of a tile
    const int log_b = 6 - log_n;           // tiles of a batch of 64
    PagedWalk<kAllRows, kTile, false, 0> walk(p.work, by_xcd(blockIdx.x, p.work.n_wg));
    while (walk.more()) {
        const PagedSeq seq = walk.seq;
        const int G = p.work.G;
        const int h = uniform(walk.h) * WAVES + wave - slot * side;
        const int rows = uniform(seq.n * G);
        const int t0 = uniform(walk.tile.first + walk.begin());
        const int nt = uniform(walk.tile.hi >= walk.tile.lo && slot < step && h < p.Hkv ? walk.count() : 0);
        i32x4_t tab_rsrc = make_rsrc_v(p.c.table + walk.b * p.c.table_s, (uint32_t)p.c.width * 4u);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            tab_rsrc[e] = uniform(tab_rsrc[e]);
        }
        // Row tiles in turn, each over the keys again.  The first has all of them, of which it reads
        // those that a row of it sees and the others' weights alone, the later ones those tiles
        // (each key's in the same wave).
        for (int base = 0; base < rows; base += kTile) {
            const bool later = base > 0;
            int key_lo, key_hi;
            visible_key_range(paged_mask(p.mask, seq), base / G, (min(base + kTile, rows) - 1) / G, key_lo, key_hi);
            key_lo = uniform(key_lo);
            key_hi = uniform(key_hi);
            const int first = t0 + (later ? max(key_lo / kTile - t0, 0) / step * step : 0) + slot;
            const int end = later ? min(t0 + nt, key_hi >= key_lo ? key_hi / kTile + 1 : 0) : t0 + nt;
            const int mine = end > first ? (end - first + step - 1) / step : 0;
            if (mine == 0) {
                continue;
            }
            auto tile_key = [&](int j) { return (first + step * j) * kTile; };
            auto issue_tab = [&](int batch) __attribute__((always_inline)) {
                const int t = (batch << log_b) + (lane >> log_n);
                const int key = tile_key(t) + ((lane & ((1 << log_n) - 1)) << p.c.lps);
                dma_load4(tab_rsrc, (uint32_t)(key >> p.c.lps) * 4u,
                          (uint32_t)uniform((int)lds_w + C::TABS + 256 * (batch & 1)));
            };
            // Of tile j: the keys' rows, and from lanes 0 - 31 their weights, from the others their
            // scales.  `w` is where the lane's key has its weight, 0 for none.
            uint64_t w = 0, w_next = 0, small = 0;
            auto find = [&](int j) __attribute__((always_inline)) {
                const int key = tile_key(j) + l32;
                const uint32_t pg = reinterpret_cast<const uint32_t*>(
                    wsm + C::TABS)[64 * ((j >> log_b) & 1) + ((j & ((1 << log_b) - 1)) << log_n) + (l32 >> p.c.lps)];
                const bool there = key < seq.len && pg < (uint32_t)p.c.pages;
                const uint64_t pe = there ? pg : 0u;
                const uint64_t off = (uint32_t)key & page_mask;
                const uint64_t row = reinterpret_cast<uint64_t>(p.c.k) + pe * (uint64_t)p.c.k_sp +
                                     off * (uint64_t)p.c.k_st + (uint64_t)h * (uint64_t)p.c.k_sh;
                rows_at[l32] = there && key >= key_lo && key <= key_hi ? row : zero;
                w_next = there ? reinterpret_cast<uint64_t>(p.w) + 4 * (pe * (uint64_t)p.w_sp + off * (uint64_t)p.w_st +
                                                                        (uint64_t)h * (uint64_t)p.w_sh)
                               : 0;
                small = g == 0 && w_next != 0 && (later || key < seq.len - seq.n) ? w_next : zero;
                if constexpr (I8) {
                    const uint64_t at = reinterpret_cast<uint64_t>(p.c.ks) +
                                        4 * (pe * (uint64_t)p.c.ks_sp + off * (uint64_t)p.c.ks_st +
                                             (uint64_t)h * (uint64_t)p.c.ks_sh);
                    small = g == 0 ? small : there ? at : zero;
                }
            };
            auto issue = [&](int j) __attribute__((always_inline)) {
                const uint32_t to = lds_w + (uint32_t)(j & 1) * C::TILE_BYTES;
                uint64_t from[C::DMA];
#pragma unroll
                for (int d = 0; d < C::DMA; d++) {
                    from[d] = *reinterpret_cast<const uint64_t*>(reinterpret_cast<const char*>(rows_at) +
                                                                 (src[d] & 0xffffu)) +
                              (src[d] >> 16);
                }
#pragma unroll
                for (int d = 0; d < C::DMA; d++) {
                    dma_gather16_nt(from[d], to + 1024 * d);
                }
                dma_gather4(small, lds_w + C::AUX + 256 * (j & 1));
            };
            issue_tab(0);
            issue_tab(1);
            __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
            find(0);
            issue(0);

            const bool valid = base + l32 < rows;
            const int tok = valid ? (base + l32) / G : 0;
            const int head = h * G + (valid ? base + l32 - tok * G : 0);
            V8 q[NS];
            {
                const char* const row = p.q + (int64_t)(seq.q0 + tok) * p.q_st + head * p.q_sh;
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    const V8 v = *reinterpret_cast<const V8*>(row + 16 * chunk_of_q<I8>(s, g));
                    q[s] = valid ? (p.q_sign < 0.0f ? -v : v) : V8{};
                }
                const RowLse r = row_lse(valid ? p.lse[(int64_t)(seq.q0 + tok) * p.Hq + head] : -INFINITY);
                rows_lse[l32] = r.sub;
                rows_lse[kTile + l32] = r.factor;
            }
            f4 sub[4], factor[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                sub[i] = *reinterpret_cast<const f4*>(rows_lse + 8 * i + 4 * g);
                factor[i] = *reinterpret_cast<const f4*>(rows_lse + kTile + 8 * i + 4 * g);
            }
            __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
            for (int j = 0; j < mine; j++) {
                w = w_next;
                if (j + 1 < mine) {
                    find(j + 1);
                    // the batch in front is done with; it lands before tile j + 1 does
                    if (((j + 1) & ((1 << log_b) - 1)) == 0) {
                        issue_tab(((j + 1) >> log_b) + 1);
                    }
                    __builtin_amdgcn_s_waitcnt(waitcnt_lgkm(0)); // every read of tile j - 1 has returned
                    issue(j + 1);
                    __builtin_amdgcn_s_waitcnt(waitcnt_vm(C::DMA + 1)); // tile j has landed
                } else {
                    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
                }
                asm volatile("" ::: "memory");
                const char* const row = wsm + (j & 1) * C::TILE_BYTES + l32 * C::RB;
                f16x s = {};
                if constexpr (I8) {
                    operand_stream<NS / 2, 4>(
                        [&](int i) { return *reinterpret_cast<const i4*>(row + (((2 * i + g) ^ swz8<D>(l32)) << 4)); },
                        [&](int i, i4 x) {
                            s = paged_mfma<T>(q[2 * i], widen_int8<T>(i2v{x[0], x[1]}), s);
                            s = paged_mfma<T>(q[2 * i + 1], widen_int8<T>(i2v{x[2], x[3]}), s);
                        });
                } else {
                    operand_stream<NS, 4>(
                        [&](int i) {
                            return *reinterpret_cast<const V8*>(row + (((2 * i + g) ^ paged_swz<D>(l32)) << 4));
                        },
                        [&](int i, V8 x) { s = paged_mfma<T>(q[i], x, s); });
                }
                const float* const aux = reinterpret_cast<const float*>(wsm + C::AUX + 256 * (j & 1));
                const float was = aux[l32];
                const float c = I8 ? p.scale_log2e * aux[kTile + l32] : p.scale_log2e;
                const int key = tile_key(j) + l32, row0 = base + 4 * g;
                const PagedKeyRows seen = paged_key_rows(p.mask, seq, G, key);
                float sum;
                if (wave_any(seen.lo > base || seen.hi < base + kTile - 1)) {
                    sum = sum_weights<true, true>(s, c, sub, factor, seen.lo - row0, seen.hi - row0, 0.0f);
                } else {
                    sum = sum_weights<false, true>(s, c, sub, factor, 0, 0, 0.0f);
                }
                sum = pair_sum(sum);
                if (g == 0 && w != 0) {
                    *reinterpret_cast<float*>(w) = later ? was + sum : new_weight(p, key < seq.len - seq.n, sum, was);
                }
            }
            __builtin_amdgcn_s_waitcnt(0); // the weights, which the next row tile reads, too
        }
        walk.next();
    }
}

template <int D, bool I8>
struct ManyCfg {
    static constexpr int WAVES = 4;
    static constexpr int THREADS = 64 * WAVES;
    // 32-key tiles in registers (us of 2 prompts of 2048 rows, 32 heads, with one less: D 64 44.6 -> 46.8,
    // D 128 61.8 -> 64.5, D 256 124 -> 181; with one more they do not fit)
    static constexpr int KT = D <= 64 ? 4 : D <= 128 ? 3 : 2;
    static constexpr int BLOCK = kTile * KT;
    static constexpr int WAVES_PER_SIMD = D <= 128 ? 2 : 1;
    // of an item beside its row tiles (us of 2 prompts of 4096 rows with 8 / 16 / 24 / 32 / 40: 214 / 197 /
    // 196 / 198 / 200)
    static constexpr int COST = 24;
    static constexpr int RB = 2 * D;
    static constexpr int KCH = D / 8;
    static constexpr int Q_BYTES = kTile * RB;
    static constexpr int NS = D / 16;
    static constexpr int LDS_BYTES = WAVES * (2 * Q_BYTES + kTile * 16); // and row addresses, log-sum-exps
    static_assert(LDS_BYTES + WAVES * BLOCK * 4 <= 160 * 1024 / (D <= 128 ? 2 : 1), "workgroups fit the LDS");
};

template <class T, int D, bool I8>
__global__ __launch_bounds__((ManyCfg<D, I8>::THREADS), (ManyCfg<D, I8>::WAVES_PER_SIMD)) void paged_weights_many(
    WeightsParams p) {
    using C = ManyCfg<D, I8>;
    using V8 = typename PagedVec<T>::v8;
    __shared__ __attribute__((aligned(16))) char dsm[C::LDS_BYTES];
    __shared__ float sums[C::WAVES][C::BLOCK];
    const int tid = threadIdx.x;
    const int wave = uniform(tid >> 6);
    const int lane = tid & 63;
    const int l32 = lane & 31, g = lane >> 5;
    const uint32_t lds_w = (uint32_t)reinterpret_cast<uintptr_t>(dsm) + wave * 2 * C::Q_BYTES;
    char* const qsm = dsm + wave * 2 * C::Q_BYTES;
    uint64_t* const rows_at = reinterpret_cast<uint64_t*>(dsm + C::WAVES * 2 * C::Q_BYTES) + wave * 2 * kTile;
    float* const lsm = reinterpret_cast<float*>(rows_at + kTile);
    const int tok_step = C::WAVES * kTile / p.work.G, head_step = C::WAVES * kTile - tok_step * p.work.G;
    uint32_t src[C::NS]; // as in paged_weights_few
#pragma unroll
    for (int n = 0; n < C::NS; n++) {
        const int c = 64 * n + lane;
        const int x = c / C::KCH;
        src[n] = (uint32_t)(x * 8) | (uint32_t)(((c - x * C::KCH) ^ paged_swz<D>(x)) * 16) << 16;
    }

    PagedItemWalk<PagedKeyItems<C::BLOCK, kTile>, true, C::COST, false> walk(p.work, by_xcd(blockIdx.x, p.work.n_wg));
    PagedRecord rec = {};
    while (walk.more()) {
        const PagedSeq seq = walk.seq;
        const int h = uniform(walk.h), G = p.work.G;
        const int rows = uniform(seq.n * G);
        const int32_t* const table = p.c.table + walk.b * p.c.table_s;
        {
            const int key0 = uniform(walk.rt) * C::BLOCK;
            // this share's of the row tiles that some key of the block is seen by
            const int rt0 = uniform(walk.tile.first + walk.begin());
            const int rt1 = uniform(walk.tile.hi >= walk.tile.lo ? rt0 + walk.count() - 1 : rt0 - 1);

            // The row of the next tile whose address this lane finds: its token and head (of the
            // group), which a step of a row tile for each wave moves on.
            int row = (rt0 + wave) * kTile + l32;
            int tok = row / G, sub_head = row - tok * G;
            float lse_next = 0.0f;
            auto prefetch = [&](int slot) __attribute__((always_inline)) {
                const bool in = row < rows; // the last row again for those behind it
                const int t = in ? tok : seq.n - 1;
                const int x = h * G + (in ? sub_head : G - 1);
                rows_at[l32] = reinterpret_cast<uint64_t>(p.q) + (uint64_t)(uint32_t)(seq.q0 + t) * (uint64_t)p.q_st +
                               (uint64_t)(uint32_t)x * (uint64_t)p.q_sh;
                lse_next = p.lse[(int64_t)(seq.q0 + t) * p.Hq + x];
                row += C::WAVES * kTile;
                tok += tok_step;
                sub_head += head_step;
                tok += sub_head >= G ? 1 : 0;
                sub_head -= sub_head >= G ? G : 0;
                uint64_t from[C::NS];
#pragma unroll
                for (int n = 0; n < C::NS; n++) {
                    from[n] = *reinterpret_cast<const uint64_t*>(reinterpret_cast<const char*>(rows_at) +
                                                                 (src[n] & 0xffffu)) +
                              (src[n] >> 16);
                }
#pragma unroll
                for (int n = 0; n < C::NS; n++) {
                    dma_gather16(from[n], (uint32_t)uniform((int)lds_w + slot * C::Q_BYTES + 1024 * n));
                }
            };
            int rt = rt0 + wave;
            int32_t entry[C::KT];
#pragma unroll
            for (int t = 0; t < C::KT; t++) {
                entry[t] = key_entry(p, seq, table, key0 + kTile * t + l32);
            }
            if (rt <= rt1) {
                prefetch(0);
            }
            KeyRegs<D, I8> raw[C::KT];
            V8 k[C::KT][C::NS];
            float scale[C::KT], sum[C::KT];
            int full_lo[C::KT], full_hi[C::KT]; // rows that see all keys of a tile
#pragma unroll
            for (int t = 0; t < C::KT; t++) {
                const int first = key0 + kTile * t;
                const LaneKey key = lane_key<I8>(p, entry[t], h, first + l32);
                raw[t].load(key.k, g);
                scale[t] = p.scale_log2e * key.k_scale * p.q_sign;
                full_lo[t] = uniform(paged_key_rows(p.mask, seq, G, min(first + kTile, seq.len) - 1).lo);
                full_hi[t] = uniform(paged_key_rows(p.mask, seq, G, first).hi);
                sum[t] = 0.0f;
            }
#pragma unroll
            for (int t = 0; t < C::KT; t++) {
#pragma unroll
                for (int s = 0; s < C::NS; s++) {
                    k[t][s] = raw[t].template operand<T>(s);
                }
            }
            for (int slot = 0; rt <= rt1; rt += C::WAVES, slot ^= 1) {
                lsm[l32] = row_lse(lse_next).sub;
                // this tile's Q has landed, and what the next one overwrites has been read
                __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
                __builtin_amdgcn_s_waitcnt(waitcnt_lgkm(0));
                asm volatile("" ::: "memory");
                if (rt + C::WAVES <= rt1) {
                    prefetch(slot ^ 1);
                }
                f4 sub[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sub[i] = *reinterpret_cast<const f4*>(lsm + 8 * i + 4 * g);
                }
                f16x acc[C::KT];
                int ln = lane; // the operands' addresses are made for every tile, not kept
                asm volatile("" : "+v"(ln));
                const int x32 = ln & 31;
                const char* const q = qsm + slot * C::Q_BYTES + x32 * C::RB;
                operand_stream<C::NS, 2>(
                    [&](int s) {
                        return *reinterpret_cast<const V8*>(q + ((chunk_of_q<I8>(s, ln >> 5) ^ paged_swz<D>(x32)) << 4));
                    },
                    [&](int s, V8 x) {
#pragma unroll
                        for (int t = 0; t < C::KT; t++) {
                            acc[t] = paged_mfma<T>(x, k[t][s], s == 0 ? f16x{} : acc[t]);
                        }
                    });
                const int base = rt * kTile;
#pragma unroll
                for (int t = 0; t < C::KT; t++) {
                    if (full_lo[t] > base || full_hi[t] < base + kTile - 1) {
                        const PagedKeyRows seen = paged_key_rows(p.mask, seq, G, key0 + kTile * t + l32);
                        const int row0 = base + 4 * g;
                        sum[t] = sum_weights<true, false>(acc[t], scale[t], sub, sub, seen.lo - row0, seen.hi - row0,
                                                          sum[t]);
                    } else {
                        sum[t] = sum_weights<false, false>(acc[t], scale[t], sub, sub, 0, 0, sum[t]);
                    }
                    __builtin_amdgcn_sched_barrier(0); // one tile's exponents in registers
                }
            }
#pragma unroll
            for (int t = 0; t < C::KT; t++) {
                const float x = pair_sum(sum[t]);
                if (g == 0) {
                    sums[wave][kTile * t + l32] = x;
                }
            }
            __syncthreads();
            if (tid < C::BLOCK) {
                float x = 0.0f;
#pragma unroll
                for (int w = 0; w < C::WAVES; w++) {
                    x += sums[w][tid];
                }
                if (walk.whole()) {
                    const int at = key0 + tid;
                    const LaneKey key = lane_key<false>(p, key_entry(p, seq, table, at), h, at);
                    const bool is_old = at < seq.len - seq.n;
                    if (key.w != nullptr) {
                        *key.w = new_weight(p, is_old, x, is_old ? *key.w : 0.0f);
                    }
                } else {
                    p.parts[(int64_t)walk.slot() * C::BLOCK + tid] = x;
                }
            }
            if (!walk.whole() && walk.begin() == 0) {
                rec = PagedRecord{C::BLOCK, walk.b, key0, h, walk.last_wg(), {}};
            }
            __syncthreads(); // before the sums of the next block
        }
        walk.next();
    }
    if (tid == 0) {
        p.records[walk.part.wg] = rec;
    }
}

// Workgroup w: the block that starts in worker w's share and goes on behind it, if there is
// one: its parts' sums, in order.
__global__ __launch_bounds__(128) void paged_weights_merge(WeightsParams p) {
    const int w = blockIdx.x;
    const PagedRecord rec = p.records[w];
    const int i = threadIdx.x;
    if (i >= rec.rows) {
        return;
    }
    const PagedSeq seq = paged_seq(p.work.seqs, rec.q0);
    const int at = rec.r0 + i;
    const LaneKey key = lane_key<false>(p, key_entry(p, seq, p.c.table + rec.q0 * p.c.table_s, at), rec.h, at);
    const bool is_old = at < seq.len - seq.n;
    const float old = key.w != nullptr && is_old ? *key.w : 0.0f;
    float sum = p.parts[(int64_t)(p.work.n_wg + w) * rec.rows + i];
    for (int s = w + 1; s <= rec.w_last; s++) {
        sum += p.parts[(int64_t)s * rec.rows + i];
    }
    if (key.w != nullptr) {
        *key.w = new_weight(p, is_old, sum, old);
    }
}

template <class T, int D, bool I8>
int launch_weights(const PagedWeightsArgs& a, WeightsParams& p, hipStream_t stream, std::string& err) {
    auto go = [&](auto* kernel, int threads, int64_t units, int min_units, int block) {
        const int64_t resident = resident_workgroups(reinterpret_cast<const void*>(kernel), threads, err);
        if (resident <= 0) {
            return -1;
        }
        p.work.min_units = min_units;
        p.work.n_wg = paged_workgroups(resident, units, min_units);
        StreamScratch ws(ScratchUse::PagedPartials);
        if (block > 0) {
            const size_t sums = (size_t)2 * p.work.n_wg * block * sizeof(float);
            if (ws.alloc(sums + p.work.n_wg * sizeof(PagedRecord), stream, err) != 0) {
                return -1;
            }
            p.parts = static_cast<float*>(ws.ptr);
            p.records = reinterpret_cast<PagedRecord*>(static_cast<char*>(ws.ptr) + sums);
        }
        hipLaunchKernelGGL(kernel, dim3((uint32_t)p.work.n_wg), dim3(threads), 0, stream, p);
        if (block > 0) {
            hipLaunchKernelGGL(paged_weights_merge, dim3((uint32_t)p.work.n_wg), dim3(128), 0, stream, p);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            err = hipGetErrorString(e);
            return -1;
        }
        return 0;
    };
    // Beyond 8 kv heads the last waves of a group of heads may be idle, which costs every row tile
    // their share: us for 32 sequences of 8192 bf16 keys of 9 heads, D 128, few / many: 64 rows 286 /
    // 372, 96 428 / 405; of 12 heads 96 512 / 551, 128 681 / 571; 16 of 9 heads, int8, 96 176 / 196,
    // 128 232 / 203.  (With fewer heads HBM is busy all the same: 5 heads, 128 rows 242 / 252.
    // Above D = 128 few is faster with idle waves too: 8 of 9 heads, D 256, 128 rows 213 / 261.)
    constexpr int W = FewCfg<D, I8>::WAVES;
    const int few_max = D > 128 || p.Hkv <= W ? kFewMax : (int)((int64_t)kFewMax * p.Hkv / ((p.Hkv + W - 1) / W * W));
    // as in paged_attention: each launch takes the sequences of its kind
    const bool any_many = (int64_t)a.max_rows_seq * p.work.G > few_max;
    const bool any_few = !any_many || a.seqs.cu != nullptr;
    PagedLaunch few, many;
    if (any_many && any_few) {
        few.max_rows = many.min_rows = few_max;
    }
    PagedWork wf = paged_work(p.work, few), wm = paged_work(p.work, many);
    wm.mask = p.mask;
    wf.Hkv = (p.Hkv + W - 1) / W;
    const int64_t cf = any_few ? paged_max_cost<kAllRows, kTile, 0>(wf) : 0;
    using C = ManyCfg<D, I8>;
    const int64_t cm = any_many ? paged_max_key_cost<C::BLOCK, kTile, C::COST>(wm) : 0;
    if (std::max(cf, cm) > INT32_MAX) {
        err = "too many rows x heads x keys that the page table covers (at most 2^31 - 1 key tiles)";
        return -1;
    }
    if (any_many) {
        p.work = wm;
        if (go(&paged_weights_many<T, D, I8>, C::THREADS, cm, 2 * C::COST, C::BLOCK) != 0) {
            return -1;
        }
    }
    if (any_few) {
        p.work = wf;
        return go(&paged_weights_few<T, D, I8>, 64 * FewCfg<D, I8>::WAVES, cf, 1, 0);
    }
    return 0;
}

} // namespace

int paged_key_weights(const PagedWeightsArgs& a, hipStream_t stream, std::string& err) {
    WeightsParams p{};
    p.c = a.c;
    p.work.seqs = a.seqs;
    p.work.mask = PagedMask{0, 0};
    p.work.Hkv = a.Hkv;
    p.work.G = a.Hq / a.Hkv;
    p.mask = a.mask;
    p.q = static_cast<const char*>(a.q);
    p.q_st = a.q_st;
    p.q_sh = a.q_sh;
    p.lse = a.lse;
    p.Hq = a.Hq;
    p.Hkv = a.Hkv;
    p.scale_log2e = softmax_log2_scale(a.scale);
    p.q_sign = a.scale < 0.0f ? -1.0f : 1.0f;
    p.decay = a.decay;
    p.w = a.w;
    p.w_sp = a.w_sp;
    p.w_st = a.w_st;
    p.w_sh = a.w_sh;
    PagedAttnArgs types; // of the kernels
    types.type = a.type;
    types.i8 = a.i8;
    types.D = a.D;
    return paged_for_type(types, [&](auto t, auto d, auto i8) {
        return launch_weights<decltype(t), decltype(d)::value, decltype(i8)::value>(a, p, stream, err);
    });
}

} // namespace rdna_amd
