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
// at a time.  6 sequences, 8 heads of 256 bytes, 256-2000 of up to 3900 keys stay, both
// launches: 26.2 us; 1024 rows at a time 25.8 (4 sequences of 600 keys 17.0 for 16.3), 256
// 26.6, 32 bytes of a row 28.5; with 512 threads 29 and, 128 bytes of a row, 32-36.
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
    for (int32_t i = lo + tid; i < min(hi, CACHE); i += kSelectThreads) {
        cache[i] = load(i);
    }
    // the smallest weight that stays, without its lowest `shift` bits (`least`), and of those equal
    // to it how many (`more`): all of them where the bits behind do not matter
    uint32_t least = 0xffffffffu;
    int shift = 0;
    if (more > 0) {
        least = 0;
        for (shift = 24;; shift -= 8) {
            if (tid < kHists * 256) {
                (&hist[0][0])[tid] = 0;
            }
            __syncthreads();
            for (int32_t i = lo + tid; i < hi; i += kSelectThreads) {
                const uint32_t u = weight(i);
                if (shift == 24 || u >> (shift + 8) == least) {
                    atomicAdd(&hist[wave % kHists][(u >> shift) & 255u], 1);
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
            least = least << 8 | (uint32_t)found[0];
            more = found[1];
            if (shift == 0 || more == found[2]) {
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

// Workgroup x, b: a slice of 64 bytes of a head's keys or values, or a head's weights.  The
// kept rows of a stretch are in registers before the first of them is written, to places
// at or before their own and behind those of every earlier stretch: later rows are not
// touched.
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
    for (int32_t r0 = 0; r0 < a.budget; r0 += PASSES * kRows) {
        i4 x[PASSES];
        float sc[PASSES];
        int32_t to[PASSES];
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const int32_t r = r0 + i * kRows + (int)threadIdx.x / LANES;
            const int32_t from = r < a.budget ? kept[r] : r;
            to[i] = -1;
            x[i] = i4{0, 0, 0, 0};
            sc[i] = 0.0f;
            if (from != r) {
                const int32_t pf = page(from);
                if (pf >= 0) {
                    to[i] = page(r);
                    const int64_t off = from & mask;
                    x[i] = *reinterpret_cast<const i4*>(base + pf * sp + off * st);
                    if (scales) {
                        sc[i] = sbase[pf * ssp + off * sst];
                    }
                }
            }
        }
        // every load has returned before any wave stores
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            asm volatile("" ::"v"(x[i]), "v"(sc[i]));
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const int32_t r = r0 + i * kRows + (int)threadIdx.x / LANES;
            if (to[i] >= 0) {
                const int64_t off = r & mask;
                *reinterpret_cast<i4*>(base + to[i] * sp + off * st) = x[i];
                if (scales) {
                    sbase[to[i] * ssp + off * sst] = sc[i];
                }
            }
        }
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
    // heads 182 us with 8192 weights and 190 with 34816; 64 x 30000 keys 456 and 307.
    auto* const choose = p.max_keys <= 8192 ? &paged_evict_choose<8192> : &paged_evict_choose<34816>;
    hipLaunchKernelGGL(choose, dim3((uint32_t)a.Hkv, (uint32_t)a.B), dim3(kSelectThreads), 0, stream, p);
    if (launched() != 0) {
        return -1;
    }
    hipLaunchKernelGGL(paged_evict_move, dim3((uint32_t)(a.Hkv * (2 * p.slices + 1)), (uint32_t)a.B), dim3(kMoveThreads), 0, stream,
                       p);
    return launched();
}

} // namespace rdna_amd
