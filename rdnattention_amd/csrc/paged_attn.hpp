// Shared by the two paged attention kernels (device code): element types, the
// walk over a workgroup's share of the work, row pointers into the pages, and
// what a shared item leaves for the merge.
#pragma once

#include "fa_common.hpp"
#include "fa_splitk.hpp"
#include "paged_host.hpp"

namespace rdna_amd {

template <class T>
struct PagedVec {
    typedef T v8 __attribute__((ext_vector_type(8)));
    typedef T v4 __attribute__((ext_vector_type(4)));
};

template <class T>
__device__ __forceinline__ f16x paged_mfma(typename PagedVec<T>::v8 a, typename PagedVec<T>::v8 b, f16x c) {
    if constexpr (sizeof(T) == 2 && __is_same(T, _Float16)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
}

// What a share of the work leaves where an item has several: slot w holds the
// part of worker w's first item that began before w, slot n_wg + w the part of
// its last item that goes on behind it (slot_rows rows: O unnormalised in fp32,
// then (m, l) with m in log2 units).  The record of worker w names the item
// that starts in it and goes on, for the merge.
struct PagedRecord {
    int32_t rows;   // 0: none
    int32_t q0;     // first token of the sequence
    int32_t r0;     // first row of the item
    int32_t h;      // kv head
    int32_t w_last; // the last worker of the item
    int32_t unused[3];
};

struct PagedAttnParams {
    PagedPages c;
    PagedWork work;
    const char* q;
    char* o;
    int64_t q_st, q_sh, o_st, o_sh; // bytes
    float scale_log2e;              // |scale| log2(e)
    float q_sign;
    int32_t zero_tail;
    int32_t Hq;
    const uint8_t* tree; // null: no tree
    int64_t tree_sb, tree_sr;
    int32_t tree_n;
    int32_t slot_rows; // rows of a slot
    float* part_o;
    float* part_ml;
    PagedRecord* records;
};

// 16-byte chunk swizzle of row r of a tile of unpadded rows (see dec_swz of the
// split-K kernel: rows that start in the same bank differ in it, so 16-row
// ds_read_b128 and 4-row transpose reads hit distinct banks).
template <int D>
__device__ __forceinline__ int paged_swz(int r) {
    if constexpr (D % 64 == 32) {
        return (r >> 2) & 3;
    } else if constexpr (D % 128 == 64) {
        return (((r >> 1) & 3) << 1) | ((r >> 3) & 1);
    } else {
        return ((r & 7) << 1) | ((r >> 3) & 1);
    }
}

// A row of zeros: stands for keys that no row of the item sees, so that what the
// pages hold there (a key behind the sequence's last may be anything) never
// meets a weight of zero as infinity or NaN.
__device__ __attribute__((aligned(16))) const uint32_t kPagedZeroRow[256 / 2] = {};

// A value that is the same in every lane, in a scalar register.
__device__ __forceinline__ int32_t uniform(int32_t x) {
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ uint64_t uniform64(uint64_t x) {
    return ((uint64_t)(uint32_t)uniform((int32_t)(x >> 32)) << 32) | (uint32_t)uniform((int32_t)(uint32_t)x);
}

// Lane x's value of all lanes.
__device__ __forceinline__ uint64_t readlane64(uint64_t v, int x) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int32_t)(v >> 32), x) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int32_t)(uint32_t)v, x);
}

// HBM -> LDS copies with a 64-bit address per lane.  The wait states are those of
// dma_load16: M0 is the only scalar register here.
__device__ __forceinline__ void dma_gather16(uint64_t addr, uint32_t lds_byte_addr) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :
                 : "v"(addr), "s"(uniform((int32_t)lds_byte_addr))
                 : "memory", "m0");
}
// ... at a wave-uniform address and 32 bits per lane.  The address usually comes straight
// from v_readlane: copied by a scalar instruction, for which the hardware waits, it needs no
// wait states before the load, and the copy is the one that M0 needs.
__device__ __forceinline__ void dma_uniform16(uint64_t base, uint32_t off, uint32_t lds_byte_addr) {
    uint64_t at;
    asm volatile("s_mov_b32 m0, %3\n\ts_mov_b64 %0, %2\n\tglobal_load_lds_dwordx4 %1, %0"
                 : "=&s"(at)
                 : "v"(off), "s"(uniform64(base)), "s"(uniform((int32_t)lds_byte_addr))
                 : "memory", "m0");
}
__device__ __forceinline__ void dma_gather16_nt(uint64_t addr, uint32_t lds_byte_addr) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt"
                 :
                 : "v"(addr), "s"(uniform((int32_t)lds_byte_addr))
                 : "memory", "m0");
}

__device__ __forceinline__ void dma_gather4(uint64_t addr, uint32_t lds_byte_addr) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
                 :
                 : "v"(addr), "s"(uniform((int32_t)lds_byte_addr))
                 : "memory", "m0");
}

typedef int i2v __attribute__((ext_vector_type(2)));

// 8 signed bytes -> T, exactly.  fp16: a byte u = v + 128 below the exponent byte of
// 1024 is 1024 + u, less 1152 it is v, five instructions per 4 values; bf16: through
// fp32, whose upper half holds all 8 bits.
template <class T>
__device__ __forceinline__ typename PagedVec<T>::v8 widen_int8(i2v w) {
    typename PagedVec<T>::v8 y;
    if constexpr (__is_same(T, _Float16)) {
        const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const uint32_t u = (uint32_t)w[c] ^ 0x80808080u;
            const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
            const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
            y[4 * c] = a[0];
            y[4 * c + 1] = a[1];
            y[4 * c + 2] = b[0];
            y[4 * c + 3] = b[1];
        }
    } else {
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        u4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t u = (uint32_t)w[i >> 1] ^ 0x80808080u;
            const float a = (float)((u >> (16 * (i & 1))) & 0xffu) - 128.0f;
            const float b = (float)((u >> (16 * (i & 1) + 8)) & 0xffu) - 128.0f;
            r[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        }
        y = __builtin_bit_cast(decltype(y), r);
    }
    return y;
}

// ds_read_b64_tr_b8: within each 16-lane group, lane i receives as byte k the byte i
// % 8 of the 8-byte word whose address lane 2k + i / 8 supplies.
__device__ __forceinline__ i2v read_tr8(const char* p) {
    typedef __attribute__((address_space(3))) i2v lds_i2;
    const auto* lp = reinterpret_cast<const __attribute__((address_space(3))) char*>(
        (uint32_t)reinterpret_cast<uintptr_t>(p));
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2*)lp);
}

// The values' scales of int8 pages, in the weights of P V: p v = (p s) (v / s), with
// p s rounded to fp16 where p would be.  So that the products keep fp16's range
// whatever the scales' size, they carry a power of two: relative to the largest
// scale so far, at 2^7 (weights reach 2^8, products 2^15); O follows when it grows.
// A value whose scale is less than 2^-21 of the largest one seen with it loses bits,
// at most 2^-32 of the largest value per key.
struct ValueScale {
    int e = -1000; // the largest scale is below 2^e

    // p[4 i + j] *= s[i][j], 2^(7 - e) times; s the scales of the lane's scores, the
    // same in each half of the wave
    template <int N, int NDT>
    __device__ __forceinline__ void weigh(float (&p)[4 * N], const f4 (&s)[N], f16x (&o)[NDT]) {
        float mx = max_tree<4 * N>([&](int i) { return fabsf(s[i >> 2][i & 3]); });
        mx = pair_max(mx);
        const int top = __builtin_amdgcn_readfirstlane(mx > 0.0f ? __builtin_amdgcn_frexp_expf(mx) : -1000);
        if (top > e) {
            const float f = ldexpf(1.0f, e - top);
#pragma unroll
            for (int i = 0; i < NDT; i++) {
                o[i] *= f;
            }
            e = top;
        }
#pragma unroll
        for (int i = 0; i < 4 * N; i++) {
            p[i] *= ldexpf(s[i >> 2][i & 3], 7 - e);
        }
    }
    __device__ __forceinline__ float factor() const {
        return ldexpf(1.0f, e - 7);
    }
};

// 16 bytes of LDS
template <class V>
__device__ __forceinline__ V lds_read(uint32_t at) {
    return *reinterpret_cast<const __attribute__((address_space(3))) V*>(at);
}
__device__ __forceinline__ h4 lds_read_tr16(uint32_t at) {
    typedef __attribute__((address_space(3))) fp16x4_raw lds_h4;
    return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                                      (lds_h4*)reinterpret_cast<const __attribute__((address_space(3))) char*>(at)));
}

// max of three, and of s[0 .. 16 N - 1]: the instruction itself, since fmaxf gets a
// canonicalising instruction in front for every operand that may be a NaN.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
template <int N>
__device__ __forceinline__ float scores_max(const f16x (&s)[N]) {
    float m[4]; // independent chains
#pragma unroll
    for (int c = 0; c < 4; c++) {
        m[c] = max3(s[0][c], s[0][4 + c], s[0][8 + c]);
    }
#pragma unroll
    for (int c = 0; c < 4; c++) {
        if constexpr (N == 1) {
            m[c] = max3(m[c], s[0][12 + c], s[0][12 + c]);
        } else {
            m[c] = max3(m[c], s[0][12 + c], s[1][c]);
        }
    }
    if constexpr (N == 2) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            m[c] = max3(m[c], s[1][4 + c], s[1][8 + c]);
        }
        m[0] = max3(m[0], s[1][12], s[1][13]);
        m[1] = max3(m[1], s[1][14], s[1][15]);
    }
    return pair_max(max3(max3(m[0], m[1], m[2]), m[3], m[3]));
}

// acc + the sum of the eight weights of v
template <class T>
__device__ __forceinline__ float sum8(typename PagedVec<T>::v8 v, float acc) {
    typedef T v2 __attribute__((ext_vector_type(2)));
    const v2 one = {(T)1.0f, (T)1.0f};
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const v2 pr = {v[e], v[e + 1]};
        if constexpr (__is_same(T, _Float16)) {
            acc = __builtin_amdgcn_fdot2(pr, one, acc, false);
        } else {
            acc = __builtin_amdgcn_fdot2_f32_bf16(pr, one, acc, false);
        }
    }
    return acc;
}

// use(j, op(j)) for j < N, op (an LDS read of an MFMA operand) DEPTH ahead of use.
// Left to itself the compiler reads each operand as it is needed and waits for it.
template <int N, int DEPTH, class Op, class Use>
__device__ __forceinline__ void operand_stream(Op&& op, Use&& use) {
    decltype(op(0)) ring[DEPTH];
#pragma unroll
    for (int j = 0; j < DEPTH && j < N; j++) {
        ring[j] = op(j);
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
        const auto a = ring[j % DEPTH];
        if (j + DEPTH < N) {
            ring[j % DEPTH] = op(j + DEPTH);
        }
        use(j, a);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Number `i` of n, where workgroup id runs on XCD id % 8, so that neighbouring numbers
// are on one XCD.
__device__ __forceinline__ int32_t by_xcd(int32_t id, int32_t n) {
    return (n & 7) == 0 ? (id & 7) * (n >> 3) + (id >> 3) : id;
}


// A worker's (a workgroup's, or a wave's) walk over its units, the same in every wave
// of it.  Sequences are counted one to a lane, and with MANY the row tiles of a longer
// one one to a lane again: one lane's count of the 64 row tiles of a prompt, three
// times over, had taken 18 us.  (Without, where a sequence is meant to have one row
// tile, longer ones are only slower.)  An item costs its units and EXTRA, the time
// before its first and after its last key tile in key tiles, and the shares are of equal
// cost: a worker with the many short row tiles at a prompt's begin has fewer key tiles.
template <int ROWS, int BN, bool MANY, int EXTRA>
struct PagedWalk {
    const PagedWork& w;
    PagedShare<EXTRA> part; // the worker's share, and of the current item
    int32_t b = 0, h = 0, rt = 0, n_rt = 0;
    PagedSeq seq;
    PagedTile tile;

    __device__ __forceinline__ PagedWalk(const PagedWork& work, int32_t worker) : w(work), part(work, uniform(worker)) {
        const int lane = threadIdx.x & 63;
        const int32_t B = w.seqs.B;
        // sequence i and what one kv head of it costs
        auto cost_of = [&](int32_t i, PagedSeq& s) {
            s = i < B ? paged_seq(w.seqs, i) : PagedSeq{0, 0, 0};
            const int32_t n = paged_row_tiles<ROWS>(w, s.n);
            int32_t u = 0;
            if (!MANY || n <= kFewTiles) {
                u = paged_head_units<ROWS, BN>(w, s) + n * EXTRA;
            }
            if constexpr (MANY) {
                for (uint64_t more = __builtin_amdgcn_ballot_w64(n > kFewTiles); more != 0; more &= more - 1) {
                    const int l = __builtin_ctzll(more);
                    const int32_t of = head_cost(PagedSeq{0, __builtin_amdgcn_readlane(s.n, l),
                                                          __builtin_amdgcn_readlane(s.len, l)});
                    u = lane == l ? of : u;
                }
            }
            return u;
        };
        // of the first 64 sequences (often all) the sums stay
        PagedSeq s0;
        const int32_t mine = cost_of(lane, s0);
        const int32_t sum = wave_prefix(mine * w.Hkv);
        int32_t total = __builtin_amdgcn_readlane(sum, 63);
        for (int32_t i = 64; i < B; i += 64) {
            PagedSeq s;
            total += __builtin_amdgcn_readlane(wave_prefix(cost_of(i + lane, s) * w.Hkv), 63);
        }
        part.deal(w, total);
        part.share = uniform(part.share);
        part.start = uniform(part.start);
        part.left = uniform(part.left);
        if (!part.more()) {
            return;
        }
        // the sequence that the share begins in
        int32_t before = 0, per_head = 0;
        for (int32_t i = 0; i < B; i += 64) {
            PagedSeq s = s0;
            int32_t m = mine, sums = sum;
            if (i > 0) {
                m = cost_of(i + lane, s);
                sums = wave_prefix(m * w.Hkv);
            }
            const uint64_t past = __builtin_amdgcn_ballot_w64(before + sums > part.start);
            if (past != 0) {
                const int l = __builtin_ctzll(past);
                b = i + l;
                per_head = __builtin_amdgcn_readlane(m, l);
                before += __builtin_amdgcn_readlane(sums, l) - per_head * w.Hkv;
                seq = PagedSeq{__builtin_amdgcn_readlane(s.q0, l), __builtin_amdgcn_readlane(s.n, l),
                               __builtin_amdgcn_readlane(s.len, l)};
                break;
            }
            before += __builtin_amdgcn_readlane(sums, 63);
        }
        b = uniform(b);
        per_head = uniform(per_head);
        if (per_head <= 0) { // (lengths that change meanwhile)
            part.left = 0;
            return;
        }
        n_rt = uniform(paged_row_tiles<ROWS>(w, seq.n));
        h = uniform(part.enter(uniform(before), per_head, w.Hkv));
        rt = 0;
        int32_t at = part.at;
        if constexpr (MANY) {
            // the row tile that `at` of the head is in
            for (int32_t first = 0; first < n_rt; first += 64) {
                const int32_t u = tile_cost(seq, n_rt, first + lane);
                const int32_t sum = wave_prefix(u);
                const uint64_t past = __builtin_amdgcn_ballot_w64(sum > at);
                if (past != 0) {
                    const int l = __builtin_ctzll(past);
                    rt = first + l;
                    at -= __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(u, l);
                    break;
                }
                at -= __builtin_amdgcn_readlane(sum, 63);
            }
            rt = uniform(rt);
            load_tile();
        } else {
            load_tile();
            while (at >= tile.units + EXTRA && rt + 1 < n_rt) {
                at -= tile.units + EXTRA;
                rt++;
                load_tile();
            }
        }
        part.at = uniform(at);
        part.item(tile.units);
    }

    static constexpr int32_t kFewTiles = 2;

    // Cost of row tile i of n.
    __device__ __forceinline__ int32_t tile_cost(const PagedSeq& s, int32_t n, int32_t i) const {
        return i < n ? paged_tile<ROWS, BN>(w, s, i).units + EXTRA : 0;
    }
    // Cost of one kv head of a sequence that is the same in every lane.
    __device__ __forceinline__ int32_t head_cost(const PagedSeq& s) const {
        const int32_t n = paged_row_tiles<ROWS>(w, s.n);
        int32_t u = 0;
        for (int32_t first = 0; first < n; first += 64) {
            u += tile_cost(s, n, first + (int)(threadIdx.x & 63));
        }
        return __builtin_amdgcn_readlane(wave_prefix(u), 63);
    }

    // Sums of x over this lane and those below it: within rows of 16 lanes by shifts,
    // then row 0's last into row 1 and row 2's into row 3, then lane 31's into the
    // upper half.
    static __device__ __forceinline__ int32_t wave_prefix(int32_t x) {
        x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true); // row_shr:1
        x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
        x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
        x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
        x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false); // row_bcast:15
        x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false); // row_bcast:31
        return x;
    }

    __device__ __forceinline__ void load_seq() {
        seq = paged_seq(w.seqs, b);
        seq.q0 = uniform(seq.q0);
        seq.n = uniform(seq.n);
        seq.len = uniform(seq.len);
        n_rt = uniform(paged_row_tiles<ROWS>(w, seq.n));
    }
    __device__ __forceinline__ void load_tile() {
        tile = paged_tile<ROWS, BN>(w, seq, rt);
        tile.lo = uniform(tile.lo);
        tile.hi = uniform(tile.hi);
        tile.first = uniform(tile.first);
        tile.units = uniform(tile.units);
    }

    // Every loop here ends by itself, whatever the lengths hold (a caller may, by
    // mistake, be changing them).
    __device__ __forceinline__ bool more() const {
        return part.more();
    }
    __device__ __forceinline__ int32_t begin() const {
        return part.begin();
    }
    __device__ __forceinline__ int32_t count() const {
        return part.count(tile.units);
    }
    __device__ __forceinline__ bool whole() const {
        return part.whole(tile.units);
    }
    __device__ __forceinline__ int32_t slot() const {
        return part.slot();
    }
    __device__ __forceinline__ int32_t last_wg() const {
        return part.last_wg(tile.units);
    }
    __device__ __forceinline__ void next() {
        part.take(tile.units);
        if (!part.more()) {
            return;
        }
        if (++rt >= n_rt) {
            rt = 0;
            if (++h == w.Hkv) {
                h = 0;
                do {
                    if (++b >= w.seqs.B) {
                        part.left = 0;
                        return;
                    }
                    load_seq();
                } while (n_rt == 0);
            }
        }
        load_tile();
        part.item(tile.units);
    }
};

// Masks the scores s[0 .. 16 N - 1] of keys key0 + 32 (e / 16) + 8 (e % 16 / 4) + e
// % 4 that row `row` of the mask (n columns, drafts from `prefix` on) does not see.
// Every byte is loaded, at a column inside the row, and then selected on: eight
// loads are in flight together.  (With the load behind the comparison this compiler, clang
// of ROCm 7.2, keeps score and result in one register and stores -inf over the
// scores that are seen.)
template <int N>
__device__ __forceinline__ void tree_mask_scores(f16x (&s)[N], const uint8_t* row, int32_t n, int32_t prefix,
                                                 int32_t key0) {
#pragma unroll
    for (int t = 0; t < 2 * N; t++) { // eight at a time: their registers
        uint32_t bit[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int32_t j = key0 + 16 * t + 8 * (e >> 2) + (e & 3) - prefix;
            bit[e] = row[max(min(j, n - 1), 0)];
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int32_t j = key0 + 16 * t + 8 * (e >> 2) + (e & 3) - prefix;
            const bool hidden = (j >= n) | ((j >= 0) & (bit[e] == 0));
            const int i = 8 * (t & 1) + e;
            s[t >> 1][i] = hidden ? -INFINITY : s[t >> 1][i];
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Zeros for the rows behind the last sequence, dealt to the workgroups.
template <int D>
__device__ __forceinline__ void zero_tail_rows(const PagedAttnParams& p) {
    constexpr int CH = D / 8;
    const int32_t per_row = p.Hq * CH;
    for (int32_t t = paged_rows_end(p.work.seqs) + blockIdx.x; t < p.work.seqs.total; t += gridDim.x) {
        for (int32_t i = threadIdx.x; i < per_row; i += blockDim.x) {
            const int32_t h = i / CH;
            *reinterpret_cast<i4*>(p.o + t * p.o_st + h * p.o_sh + 16 * (i - h * CH)) = i4{0, 0, 0, 0};
        }
    }
}

} // namespace rdna_amd
