// Eviction from a paged key/value cache: of every sequence with more keys than the
// budget, each kv head keeps the first ones, the newest ones and, of those between, the
// ones of the largest weights (equal ones: those in front), in their order.  They move up
// to the front with their values, scales and weights.
//
// Two launches.  The choice reads a head's weights once, into LDS as far as they fit, and
// finds the smallest weight that stays eight bits at a time; bound by the latency of its
// passes.  The moves read and write each kept byte once.
#include "fa_common.hpp"
#include "paged_host.hpp"

namespace rdna_amd {
namespace {

constexpr int kSelectThreads = 1024;
constexpr int kWaves = kSelectThreads / 64;
// A workgroup of moves has 64 bytes of a row (the narrowest rows are that long) and 512 rows
// at a time, and the next ones on their way.  64 sequences of 3900 keys, 8 heads of 256 bytes,
// 1000 stay, both launches: 146 us; one stretch at a time 162; 256 rows at a time 158, 1024
// 182, 32 bytes of a row 181, 512 threads 152.  2 x 8120 int8 keys, of which 7267 stay: 64 us;
// 69, 70, 60, 54, 72.
constexpr int kMoveThreads = 1024;
constexpr int kMoveLanes = 4, kMovePasses = 2;
constexpr int kHists = 4; // copies of the histogram

struct EvictParams {
    PagedEvictArgs a;
    int32_t max_keys;
    int32_t slices; // of a row
};

// Weights in an order of whole numbers: NaN below all, the zeros alike.
__device__ __forceinline__ uint32_t ordered(float w) {
    const uint32_t b = __float_as_uint(w + 0.0f);
    return w != w ? 0u : (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}

// Workgroup h, b.  CACHE: weights in LDS, those behind are read again in every pass.
template <int CACHE>
__global__ __launch_bounds__(kSelectThreads) void paged_evict_choose(EvictParams p) {
    __shared__ uint32_t cache[CACHE];
    __shared__ int32_t hist[kHists][256];
    __shared__ int32_t found[3];
    __shared__ uint32_t ends[2][kWaves];
    __shared__ int32_t counts[2][kWaves];
    const PagedEvictArgs& a = p.a;
    const int h = blockIdx.x, b = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t len = rows_clamp(a.lens[b], 0, p.max_keys);
    int32_t* const kept = a.kept + ((int64_t)b * a.Hkv + h) * a.budget;
    const int32_t n = min(len, a.budget);
    if (h == 0 && tid == 0) {
        a.new_lens[b] = n;
    }
    if (len <= a.budget) {
        for (int32_t i = tid; i < a.budget; i += kSelectThreads) {
            kept[i] = i < len ? i : -1;
        }
        return;
    }
    const int32_t* const table = a.c.table + b * a.c.table_s;
    const int32_t mask = (1 << a.c.lps) - 1;
    auto load = [&](int32_t key) {
        const int32_t pg = paged_page(a.c, table, key >> a.c.lps);
        return pg >= 0 ? ordered(a.w[pg * a.w_sp + (int64_t)(key & mask) * a.w_st + h * a.w_sh]) : 0u;
    };
    auto weight = [&](int32_t key) { return key < CACHE ? cache[key] : load(key); };
    // between the first and the newest: 0 < more <= lo .. hi's number where any of them stay
    const int32_t lo = a.first, hi = len - a.recent;
    int32_t more = a.budget - a.first - a.recent;
    uint32_t low = 0xffffffffu, high = 0;
    constexpr int NB = 4; // loads in flight: 64 x 30000 keys 276 -> 272 us
    for (int32_t i0 = lo + tid; i0 < hi; i0 += NB * kSelectThreads) {
        int32_t pg[NB];
        float w[NB];
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int32_t i = i0 + j * kSelectThreads;
            pg[j] = i < hi ? paged_page(a.c, table, i >> a.c.lps) : -1;
        }
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int32_t i = i0 + j * kSelectThreads;
            w[j] = pg[j] >= 0 ? a.w[pg[j] * a.w_sp + (int64_t)(i & mask) * a.w_st + h * a.w_sh] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const int32_t i = i0 + j * kSelectThreads;
            if (i < hi) {
                const uint32_t u = pg[j] >= 0 ? ordered(w[j]) : 0u;
                if (i < CACHE) {
                    cache[i] = u;
                }
                low = min(low, u);
                high = max(high, u);
            }
        }
    }
    // the smallest weight that stays, without its lowest `shift` bits (`least`), and of those equal
    // to it how many (`more`): all of them where the bits behind do not matter
    uint32_t least = 0xffffffffu;
    int shift = 0;
    if (more > 0) {
        // The digits begin at the first bit in which two weights differ: at bit 31 most weights of
        // a softmax would have one of two or three digits, and their atomics take turns.  One
        // sequence of 8000 keys 27.9 -> 25.9 us, of 30000 66.9 -> 59.9.
        for (int d = 1; d < 64; d <<= 1) {
            low = min(low, (uint32_t)__shfl_xor((int32_t)low, d));
            high = max(high, (uint32_t)__shfl_xor((int32_t)high, d));
        }
        if (lane == 0) {
            ends[0][wave] = low;
            ends[1][wave] = high;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            low = min(low, ends[0][w]);
            high = max(high, ends[1][w]);
        }
        shift = 32 - __builtin_clz((low ^ high) | 1u);
        least = (uint32_t)((uint64_t)high >> shift);
        for (bool all = true; shift > 0; all = false) {
            const int bits = min(8, shift);
            const int from = shift;
            shift -= bits;
            if (tid < kHists * 256) {
                (&hist[0][0])[tid] = 0;
            }
            __syncthreads();
            for (int32_t i = lo + tid; i < hi; i += kSelectThreads) {
                const uint32_t u = weight(i);
                if (all || u >> from == least) {
                    atomicAdd(&hist[wave % kHists][(u >> shift) & ((1u << bits) - 1)], 1);
                }
            }
            __syncthreads();
            if (wave == 0) {
                // lane i has digits 255 - 4 i and below
                int32_t c[4], sum = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    c[j] = 0;
#pragma unroll
                    for (int w = 0; w < kHists; w++) {
                        c[j] += hist[w][255 - 4 * lane - j];
                    }
                    sum += c[j];
                }
                int32_t above = sum; // of this lane and those below it
                for (int d = 1; d < 64; d <<= 1) {
                    const int32_t x = __shfl_up(above, d);
                    above += lane >= d ? x : 0;
                }
                above -= sum;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (above < more && more <= above + c[j]) {
                        found[0] = 255 - 4 * lane - j;
                        found[1] = more - above;
                        found[2] = c[j];
                    }
                    above += c[j];
                }
            }
            __syncthreads();
            least = least << bits | (uint32_t)found[0];
            more = found[1];
            if (more == found[2]) {
                break;
            }
        }
    }
    __syncthreads();
    // Each wave has a stretch of the keys: it counts those that stay, then the stretches in
    // front are known and it lists them.
    const int32_t part = ((len + kWaves - 1) / kWaves + 63) / 64 * 64;
    const int32_t from = min((int64_t)wave * part, (int64_t)len), to = min((int64_t)from + part, (int64_t)len);
    auto visit = [&](auto&& use) {
        for (int32_t i0 = from; i0 < to; i0 += 64) {
            const int32_t i = i0 + lane;
            const bool in = i < to;
            const bool between = in && i >= lo && i < hi;
            const uint32_t u = between ? weight(i) >> shift : 0u;
            const bool equal = between && u == least;
            use(i, __builtin_amdgcn_ballot_w64(in && (!between || u > least)), __builtin_amdgcn_ballot_w64(equal));
        }
    };
    int32_t sure = 0, ties = 0;
    visit([&](int32_t, uint64_t s, uint64_t t) {
        sure += __popcll(s);
        ties += __popcll(t);
    });
    if (lane == 0) {
        counts[0][wave] = sure;
        counts[1][wave] = ties;
    }
    __syncthreads();
    int32_t before = 0, ties_before = 0;
    for (int w = 0; w < wave; w++) {
        before += counts[0][w];
        ties_before += counts[1][w];
    }
    visit([&](int32_t i, uint64_t s, uint64_t t) {
        const uint64_t below = (1ull << lane) - 1;
        const int32_t t_here = ties_before + __popcll(t & below);
        const int32_t at = before + __popcll(s & below) + min(t_here, more);
        const bool stays = (s >> lane & 1) != 0 || ((t >> lane & 1) != 0 && t_here < more);
        if (stays && at < a.budget) { // (weights that change meanwhile)
            kept[at] = i;
        }
        before += __popcll(s);
        ties_before += __popcll(t);
    });
}

// Workgroup x, b: a slice of 64 bytes of a head's keys or values, or a head's weights.  A
// stretch of kept rows is written when it and all rows in front are in registers, to places
// at or before their own and behind those of every earlier stretch: rows of later stretches,
// already on their way, lie behind all places written so far.
__global__ __launch_bounds__(kMoveThreads) void paged_evict_move(EvictParams p) {
    constexpr int PASSES = kMovePasses, LANES = kMoveLanes;
    const PagedEvictArgs& a = p.a;
    const int b = blockIdx.y;
    const int32_t len = rows_clamp(a.lens[b], 0, p.max_keys);
    if (len <= a.budget) {
        return;
    }
    const int32_t* const table = a.c.table + b * a.c.table_s;
    const int32_t mask = (1 << a.c.lps) - 1;
    const int rows = 2 * a.Hkv * p.slices;
    const bool weights = (int)blockIdx.x >= rows;
    // the slices of a row on one XCD where the number of heads lets them
    const int slice = weights ? 0 : blockIdx.x / (2 * a.Hkv);
    const int hv = weights ? 0 : blockIdx.x % (2 * a.Hkv);
    const int h = weights ? blockIdx.x - rows : hv >> 1;
    const bool keys = (hv & 1) == 0;
    const int32_t* const kept = a.kept + ((int64_t)b * a.Hkv + h) * a.budget;
    auto page = [&](int32_t key) {
        return key >= 0 && key < p.max_keys ? paged_page(a.c, table, key >> a.c.lps) : -1;
    };
    if (weights) {
        float* const base = a.w + h * a.w_sh;
        for (int32_t r0 = 0; r0 < a.budget; r0 += PASSES * kMoveThreads) {
            float x[PASSES];
            int32_t to[PASSES];
#pragma unroll
            for (int i = 0; i < PASSES; i++) {
                const int32_t r = r0 + i * kMoveThreads + threadIdx.x;
                const int32_t from = r < a.budget ? kept[r] : r;
                to[i] = -1;
                x[i] = 0.0f;
                if (from != r) {
                    const int32_t pf = page(from);
                    if (pf >= 0) {
                        to[i] = page(r);
                        x[i] = base[pf * a.w_sp + (int64_t)(from & mask) * a.w_st];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < PASSES; i++) {
                asm volatile("" ::"v"(x[i]));
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PASSES; i++) {
                const int32_t r = r0 + i * kMoveThreads + threadIdx.x;
                if (to[i] >= 0) {
                    base[to[i] * a.w_sp + (int64_t)(r & mask) * a.w_st] = x[i];
                }
            }
        }
        return;
    }
    const int ch = threadIdx.x & (LANES - 1);
    constexpr int kRows = kMoveThreads / LANES;
    char* const base = (keys ? a.c.k + h * a.c.k_sh : a.c.v + h * a.c.v_sh) + 16 * (LANES * slice + ch);
    float* const sbase = keys ? a.c.ks + h * a.c.ks_sh : a.c.vs + h * a.c.vs_sh;
    const int64_t sp = keys ? a.c.k_sp : a.c.v_sp, st = keys ? a.c.k_st : a.c.v_st;
    const int64_t ssp = keys ? a.c.ks_sp : a.c.vs_sp, sst = keys ? a.c.ks_st : a.c.vs_st;
    const bool scales = a.i8 && slice == 0 && ch == 0;
    // Stretch s is written while the rows of s + 1 are loaded, the pages of s + 2 and the
    // numbers of s + 3.
    struct Stretch {
        i4 x[PASSES];
        float sc[PASSES];
        int32_t from[PASSES], pf[PASSES], pt[PASSES];
    };
    const int32_t row = (int32_t)threadIdx.x / LANES;
    auto number = [&](Stretch& t, int32_t s) {
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const int32_t r = (s * PASSES + i) * kRows + row;
            t.from[i] = r < a.budget ? kept[r] : r;
        }
    };
    auto find = [&](Stretch& t, int32_t s) {
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const int32_t r = (s * PASSES + i) * kRows + row;
            const bool moves = t.from[i] != r;
            t.pf[i] = moves ? page(t.from[i]) : -1;
            t.pt[i] = moves ? page(r) : -1;
        }
    };
    auto load = [&](Stretch& t) {
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            t.x[i] = i4{0, 0, 0, 0};
            t.sc[i] = 0.0f;
            if (t.pf[i] >= 0) {
                const int64_t off = t.from[i] & mask;
                t.x[i] = *reinterpret_cast<const i4*>(base + t.pf[i] * sp + off * st);
                if (scales) {
                    t.sc[i] = sbase[t.pf[i] * ssp + off * sst];
                }
            }
        }
    };
    auto step = [&](int32_t s, Stretch& now, Stretch& next, Stretch& third, Stretch& fourth) {
        load(next);
        find(third, s + 2);
        number(fourth, s + 3);
        // every wave's rows up to this stretch's are in registers before any is written
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            asm volatile("" ::"v"(now.x[i]), "v"(now.sc[i]) : "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const int32_t r = (s * PASSES + i) * kRows + row;
            if (now.pf[i] >= 0 && now.pt[i] >= 0) {
                const int64_t off = r & mask;
                *reinterpret_cast<i4*>(base + now.pt[i] * sp + off * st) = now.x[i];
                if (scales) {
                    sbase[now.pt[i] * ssp + off * sst] = now.sc[i];
                }
            }
        }
    };
    Stretch t0, t1, t2, t3;
    number(t0, 0);
    number(t1, 1);
    number(t2, 2);
    find(t0, 0);
    find(t1, 1);
    load(t0);
    const int32_t n = (a.budget + PASSES * kRows - 1) / (PASSES * kRows);
    for (int32_t s = 0; s < n; s += 4) { // places from the budget on do not move
        step(s, t0, t1, t2, t3);
        step(s + 1, t1, t2, t3, t0);
        step(s + 2, t2, t3, t0, t1);
        step(s + 3, t3, t0, t1, t2);
    }
}

} // namespace

int paged_evict(const PagedEvictArgs& a, hipStream_t stream, std::string& err) {
    EvictParams p;
    p.a = a;
    p.max_keys = (int32_t)((int64_t)a.c.width << a.c.lps);
    p.slices = a.row_bytes / (16 * kMoveLanes);
    auto launched = [&]() {
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            err = hipGetErrorString(e);
            return -1;
        }
        return 0;
    };
    // 34816 weights are nearly all LDS, so that a CU has one workgroup: 64 x 8000 keys of 8
    // heads 182 us with 8192 weights and 190 with 34816; 64 x 30000 keys 456 and 307 (both
    // before the moves overlapped their stretches).
    auto* const choose = p.max_keys <= 8192 ? &paged_evict_choose<8192> : &paged_evict_choose<34816>;
    hipLaunchKernelGGL(choose, dim3((uint32_t)a.Hkv, (uint32_t)a.B), dim3(kSelectThreads), 0, stream, p);
    if (launched() != 0) {
        return -1;
    }
    hipLaunchKernelGGL(paged_evict_move, dim3((uint32_t)(a.Hkv * (2 * p.slices + 1)), (uint32_t)a.B),
                       dim3(kMoveThreads), 0, stream, p);
    return launched();
}

} // namespace rdna_amd
