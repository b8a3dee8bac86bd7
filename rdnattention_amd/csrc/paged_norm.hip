// The append of a paged key/value cache with norms: each head of the queries and
// keys is divided by the root mean square of its channels and weighted, y = x w /
// sqrt(mean(x^2) + eps), then rotated by one position or, column by column of the
// tables, by one of several, and rounded once; keys go to their places in the
// pages, quantised where those are int8.
//
// Every byte moves once: a large call is bound by HBM, a decode step's by its chain
// of dependent loads (row range, length, page and position, angles) and the launch.
#include "fa_common.hpp"
#include "paged_host.hpp"

#include <algorithm>
#include <type_traits>

namespace rdna_amd {
namespace {

constexpr int kThreads = 256;

// Mean squares (with eps) that fp32 holds: squares below its normal range, off by up to 2^-150
// each, are 2^-50 of the least at most, and above the most the sum is infinite.  bf16 rows can
// be smaller or larger.
constexpr float kLeastMean = 0x1p-100f, kMostMean = 0x1.fffffep127f;

typedef int8_t b8 __attribute__((ext_vector_type(8)));

template <class F>
__device__ __forceinline__ F from_lane(F v, int lane) {
    if constexpr (sizeof(F) == 8) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * lane, (int)(uint32_t)u);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * lane, (int)(uint32_t)(u >> 32));
        return __builtin_bit_cast(F, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(F, __builtin_amdgcn_ds_bpermute(4 * lane, __builtin_bit_cast(int, v)));
    }
}

// Sum over a group of LANES lanes, in all of them.
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
    // neighbours and pairs within quads, then mirrored halves of 8 and 16 lanes
#define RDNA_DPP(x, ctrl) __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), ctrl, 0xf, 0xf, true))
    v += RDNA_DPP(v, 0xb1);
    v += RDNA_DPP(v, 0x4e);
    if constexpr (LANES >= 8) {
        v += RDNA_DPP(v, 0x141);
    }
    if constexpr (LANES >= 16) {
        v += RDNA_DPP(v, 0x140);
    }
#undef RDNA_DPP
    if constexpr (LANES == 32) {
        v += from_lane(v, (int)(threadIdx.x & 63) ^ 16);
    }
    return v;
}
template <int LANES>
__device__ __forceinline__ double group_sum(double v) {
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) {
        v += from_lane(v, (int)(threadIdx.x & 63) ^ d);
    }
    return v;
}

// Eight channels from chunk c of a norm's weights.
__device__ __forceinline__ void load_weights(const void* w, PagedNormType type, int c, float (&out)[8]) {
    if (type == PagedNormType::F32) {
        const f4 lo = reinterpret_cast<const f4*>(w)[2 * c], hi = reinterpret_cast<const f4*>(w)[2 * c + 1];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            out[e] = lo[e];
            out[4 + e] = hi[e];
        }
    } else if (type == PagedNormType::F16) {
        const h8 v = reinterpret_cast<const h8*>(w)[c];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            out[e] = (float)v[e];
        }
    } else {
        typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
        const bf8 v = reinterpret_cast<const bf8*>(w)[c];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            out[e] = (float)v[e];
        }
    }
}

struct NormParams {
    PagedAppendArgs a;
    PagedNorm n;
    uint32_t per_token; // groups of lanes that a token has
    uint32_t groups;    // of the call
    float inv_d;
};

template <class F>
struct Wide {
    typedef F v8 __attribute__((ext_vector_type(8)));
};

// A head x, and eps, by a power of two such that the larger of |x| and sqrt(eps) is near 1: the
// mean square and eps.
template <int LANES>
__device__ __forceinline__ float in_range(float (&x)[8], const NormParams& p) {
    float mx = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        mx = fmaxf(mx, fabsf(x[e]));
    }
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) {
        mx = fmaxf(mx, from_lane(mx, (int)(threadIdx.x & 63) ^ d));
    }
    int by = mx > 0.0f ? -__builtin_amdgcn_frexp_expf(mx) : 1000;
    by = min(by, p.n.eps > 0.0f ? -(__builtin_amdgcn_frexp_expf(p.n.eps) >> 1) : by);
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = ldexpf(x[e], by);
        sum = fmaf(x[e], x[e], sum);
    }
    return fmaf(group_sum<LANES>(sum), p.inv_d, ldexpf(p.n.eps, 2 * by));
}

// The angles of a lane's channels: of the pairs (2i, 2i + 1) four columns, of the
// halves eight.
struct Angles {
    float c[8], s[8];
};

// LANES lanes, a power of two that holds a head's D / 8 chunks of 16 bytes, have every
// per_token'th head of one token, of its keys', values' and queries'.  They look the
// token's place and angles up once (with several axes 32 loads for a head's one), and
// work on BATCH heads while the next are loaded.
template <class T, bool I8, int LANES, int BATCH>
__global__ __launch_bounds__(kThreads) void paged_append_normed(NormParams p) {
    typedef T V8 __attribute__((ext_vector_type(8)));
    const PagedAppendArgs& a = p.a;
    const uint32_t idx = (blockIdx.x * kThreads + threadIdx.x) / LANES;
    const bool live = idx < p.groups;
    const uint32_t at = live ? idx : p.groups - 1;
    const int32_t t = (int32_t)(at / p.per_token);
    const int32_t h0 = (int32_t)(at - (uint32_t)t * p.per_token);
    const int lane = threadIdx.x & 63;
    const int c = lane & (LANES - 1);
    const bool chunk = 8 * c < a.D;
    const int heads = 2 * a.Hkv + a.Hq;

    const int per = (int)p.per_token;
    auto load = [&](V8 (&x)[BATCH], int first) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            int h = min(first + i * per, heads - 1);
            const int which = h < a.Hkv ? 0 : h < 2 * a.Hkv ? 1 : 2; // keys, values, queries
            h -= which * a.Hkv;
            const char* src = which == 0   ? (const char*)a.k + t * a.k_st + h * a.k_sh
                              : which == 1 ? (const char*)a.v + t * a.v_st + h * a.v_sh
                                           : (const char*)a.q + t * a.q_st + h * a.q_sh;
            x[i] = chunk ? *reinterpret_cast<const V8*>(src + 16 * c) : V8{};
        }
    };
    V8 x[BATCH];
    load(x, h0);

    // the row's sequence and its place there (as in paged_append_rows)
    int32_t b, key;
    if (a.seqs.cu == nullptr) {
        b = paged_seq_of_row(a.seqs, t);
        key = rows_clamp(a.seqs.lens[b], 0, a.seqs.max_keys) - a.seqs.rows + (t - b * a.seqs.rows);
    } else {
        const int32_t t0 = __builtin_amdgcn_readfirstlane(t);
        b = 0;
        for (int32_t i = 0; i < a.seqs.B; i += 64) {
            const bool ended = i + lane < a.seqs.B && a.seqs.cu[i + lane + 1] <= t0;
            b += __popcll(__builtin_amdgcn_ballot_w64(ended));
        }
        b = paged_seq_of_row(a.seqs, t, b);
        key = -1;
        if (b >= 0) {
            const PagedSeq s = paged_seq(a.seqs, b);
            key = s.len - s.n + (t - s.q0);
        }
    }
    const int32_t page = key >= 0 ? paged_page(a.c, a.c.table + b * a.c.table_s, key >> a.c.lps) : -1;
    const int32_t off = key & ((1 << a.c.lps) - 1);

    const bool turns = a.rot != 0 && b >= 0 && (a.positions != nullptr || key >= 0);
    const bool mine = turns && 8 * c < a.rot; // this lane's channels are rotated
    const int half = a.rot / 2;
    const bool second = !a.interleaved && 8 * c >= half;
    const int partner = a.interleaved || !mine ? lane : second ? lane - half / 8 : lane + half / 8;
    Angles ang = {};
    if (mine) {
        const int col = a.interleaved ? 4 * c : 8 * c - (second ? half : 0);
        if (p.n.rot_axes == nullptr) {
            const int32_t pos =
                rows_clamp(a.positions != nullptr ? a.positions[t * p.n.position_s] : key, 0, a.rot_rows - 1);
            const int64_t row = (int64_t)pos * half + col;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (i == 0 || !a.interleaved) {
                    const f4 cs = *reinterpret_cast<const f4*>(a.cos + row + 4 * i);
                    const f4 sn = *reinterpret_cast<const f4*>(a.sin + row + 4 * i);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        ang.c[4 * i + e] = cs[e];
                        ang.s[4 * i + e] = sn[e];
                    }
                }
            }
        } else {
            const int32_t* const pos = a.positions + t * p.n.position_s;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (e < 4 || !a.interleaved) {
                    const int32_t axis = rows_clamp(p.n.rot_axes[col + e], 0, p.n.axes - 1);
                    const int64_t row = (int64_t)rows_clamp(pos[axis], 0, a.rot_rows - 1) * half + col + e;
                    ang.c[e] = a.cos[row];
                    ang.s[e] = a.sin[row];
                }
            }
        }
    }

    // x normed (with weights) and rotated, in F, rounded to T
    auto turned = [&](V8 v, const void* weights, auto as) __attribute__((always_inline)) -> V8 {
        using F = decltype(as);
        F y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            y[e] = (F)(float)v[e];
        }
        if (weights != nullptr && b >= 0) {
            F sum = F(0);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                sum += y[e] * y[e];
            }
            sum = group_sum<LANES>(sum);
            F r;
            if constexpr (sizeof(F) == 8) {
                r = F(1) / __builtin_elementwise_sqrt(sum / (F)a.D + (F)p.n.eps);
            } else {
                float mean = fmaf(sum, p.inv_d, p.n.eps);
                if (!(mean >= kLeastMean && mean <= kMostMean)) { // the lanes of a head are of one mind
                    mean = in_range<LANES>(y, p);
                }
                r = __builtin_amdgcn_rsqf(mean); // good to 2^-23 itself
            }
            float w[8];
            load_weights(weights, p.n.type, chunk ? c : 0, w);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[e] = y[e] * r * (F)w[e];
            }
        }
        if (a.rot == 0) {
            return __builtin_convertvector((typename Wide<F>::v8){y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]}, V8);
        }
        F z[8];
        if (a.interleaved) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                z[2 * e] = y[2 * e] * (F)ang.c[e] - y[2 * e + 1] * (F)ang.s[e];
                z[2 * e + 1] = y[2 * e] * (F)ang.s[e] + y[2 * e + 1] * (F)ang.c[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const F o = from_lane(y[e], partner);
                z[e] = y[e] * (F)ang.c[e] + o * (second ? (F)ang.s[e] : -(F)ang.s[e]);
            }
        }
        V8 r;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            r[e] = (T)(mine ? z[e] : y[e]);
        }
        return r;
    };

    for (int first = h0; first < heads; first += BATCH * per) {
        V8 now[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            now[i] = x[i];
        }
        if (first + BATCH * per < heads) {
            load(x, first + BATCH * per);
        }
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            int h = first + i * per;
            const bool has = live && h < heads; // else the last head again, for its lanes' sake
            h = min(h, heads - 1);
            const int which = h < a.Hkv ? 0 : h < 2 * a.Hkv ? 1 : 2;
            h -= which * a.Hkv;
            // Every lane of a head's group takes the same branches; what the groups of a
            // wave exchange stays within each.
            V8 y = now[i];
            if (which != 1) {
                const void* w = which == 0 ? p.n.key : p.n.query;
                if (I8 && which == 0) {
                    // keys that are quantised: in fp64, so that the row before is the nearest one
                    // and a value at a border of two int8 steps falls the way of the definition
                    y = turned(y, w, double{});
                } else {
                    y = turned(y, w, float{});
                }
            }
            if (which == 2) {
                if (has && chunk) {
                    *reinterpret_cast<V8*>((char*)a.q_out + t * a.qo_st + h * a.qo_sh + 16 * c) = y;
                }
                continue;
            }
            float scale = 0.0f;
            if constexpr (I8) {
                float mx = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float v = fabsf((float)y[e]);
                    mx = v > mx || v != v ? v : mx;
                }
#pragma unroll
                for (int d = 1; d < LANES; d <<= 1) {
                    const float v = from_lane(mx, lane ^ d);
                    mx = v > mx || v != v ? v : mx;
                }
                scale = mx * (1.0f / 127.0f);
                scale = scale == 0.0f ? 1.0f : scale;
            }
            if (page < 0 || !has || !chunk) {
                continue;
            }
            char* const dst = which == 0 ? a.c.k + page * a.c.k_sp + off * a.c.k_st + h * a.c.k_sh
                                         : a.c.v + page * a.c.v_sp + off * a.c.v_st + h * a.c.v_sh;
            if constexpr (I8) {
                b8 q;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    q[e] = (int8_t)fminf(fmaxf(rintf((float)y[e] / scale), -127.0f), 127.0f);
                }
                *reinterpret_cast<b8*>(dst + 8 * c) = q;
                if (c == 0) {
                    float* const sc = which == 0 ? a.c.ks + page * a.c.ks_sp + off * a.c.ks_st + h * a.c.ks_sh
                                                 : a.c.vs + page * a.c.vs_sp + off * a.c.vs_st + h * a.c.vs_sh;
                    *sc = scale;
                }
            } else {
                *reinterpret_cast<V8*>(dst + 16 * c) = y;
            }
        }
    }
}

template <class T, bool I8, int LANES, int BATCH>
void launch(NormParams& p, uint32_t per_token, hipStream_t stream) {
    p.per_token = per_token;
    p.groups = (uint32_t)p.a.seqs.total * p.per_token;
    const uint32_t per_block = kThreads / LANES;
    hipLaunchKernelGGL((paged_append_normed<T, I8, LANES, BATCH>), dim3((p.groups + per_block - 1) / per_block),
                       dim3(kThreads), 0, stream, p);
}

} // namespace

int paged_append_norm(const PagedAppendArgs& a, const PagedNorm& n, hipStream_t stream, std::string& err) {
    NormParams p;
    p.a = a;
    p.n = n;
    p.inv_d = 1.0f / (float)a.D;
    // Groups per token: as many as it takes for 1024 lanes (of 2048) on each of the chip's 256
    // compute units, up to one for each head, and the groups of a wave at least.  us for 4853
    // bf16 rows of 32 + 16 heads of 128 with three axes: 37 with 3 heads at a time, 38 with 2, 43
    // with 1, 50 with 4 (more than the 96 registers of five waves on a SIMD); 50 with 2048 lanes.
    const int64_t heads = 2 * a.Hkv + a.Hq;
    auto go = [&](auto t, auto i8, auto lanes_of) {
        using T = decltype(t);
        constexpr bool I8 = decltype(i8)::value;
        constexpr int L = decltype(lanes_of)::value;
        const int64_t want = std::max<int64_t>((256 * 1024) / ((int64_t)a.seqs.total * L), 64 / L);
        const uint32_t per = (uint32_t)std::min(want, heads);
        per * 2 > heads ? launch<T, I8, L, 1>(p, (uint32_t)heads, stream) : launch<T, I8, L, 3>(p, per, stream);
    };
    auto typed = [&](auto t) {
        if (a.i8) {
#if !defined(RDNATTENTION_NO_INT8)
            a.D == 64 ? go(t, std::true_type{}, std::integral_constant<int, 8>{})
                      : go(t, std::true_type{}, std::integral_constant<int, 16>{});
#endif
        } else if (a.D <= 32) {
            go(t, std::false_type{}, std::integral_constant<int, 4>{});
        } else if (a.D <= 64) {
            go(t, std::false_type{}, std::integral_constant<int, 8>{});
        } else if (a.D <= 128) {
            go(t, std::false_type{}, std::integral_constant<int, 16>{});
        } else {
            go(t, std::false_type{}, std::integral_constant<int, 32>{});
        }
    };
    a.type == PagedType::F16 ? typed(_Float16{}) : typed(__bf16{});
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        err = hipGetErrorString(e);
        return -1;
    }
    return 0;
}

} // namespace rdna_amd
