// Host check of rdnattention_amd/csrc/paged_rows.hpp: what the device code
// derives from lengths and row ranges of any content stays in bounds, and the
// units of a call cover every visible (row, key) pair.
#include "paged_rows.hpp"

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>

using namespace rdna_amd;

static long checks = 0;
static uint64_t state = 88172645463325252ull;
static uint32_t rnd() {
    state ^= state << 13;
    state ^= state >> 7;
    state ^= state << 17;
    return (uint32_t)(state >> 16);
}
static int32_t pick(int32_t lo, int32_t hi) {
    return lo + (int32_t)(rnd() % (uint32_t)(hi - lo + 1));
}
#define CHECK(x)                                                    \
    do {                                                            \
        checks++;                                                   \
        if (!(x)) {                                                 \
            std::printf("line %d: %s (case %ld)\n", __LINE__, #x, n); \
            std::exit(1);                                           \
        }                                                           \
    } while (0)

template <int ROWS, int BN>
static void one(long n) {
    const int32_t B = pick(1, 6);
    const bool ragged = rnd() % 2;
    const bool wild = rnd() % 4 == 0;
    std::vector<int32_t> lens(B), cu(B + 1);
    PagedWork w{};
    w.G = pick(1, 9);
    w.Hkv = pick(1, 3);
    w.seqs.max_keys = pick(0, 300);
    w.seqs.rows = pick(1, 40);
    int32_t at = 0;
    for (int32_t b = 0; b < B; b++) {
        cu[b] = at;
        at += pick(0, 60);
        lens[b] = wild ? (int32_t)rnd() : pick(0, w.seqs.max_keys);
    }
    cu[B] = at;
    w.seqs.total = ragged ? at + pick(0, 5) : B * w.seqs.rows;
    if (wild) {
        for (auto& x : cu) {
            x = rnd() % 3 == 0 ? (int32_t)rnd() : pick(-5, w.seqs.total + 5);
        }
    }
    w.seqs.lens = lens.data();
    w.seqs.cu = ragged ? cu.data() : nullptr;
    w.seqs.B = B;
    w.mask.causal = rnd() % 2;
    w.mask.window = rnd() % 2 ? 0 : (rnd() % 8 == 0 ? (1 << 30) - 1 : pick(1, 200));
    w.min_rows = 0;
    w.max_rows = INT32_MAX;
    w.n_wg = pick(1, 64);
    w.min_units = pick(1, 8);

    int64_t total = 0;
    for (int32_t b = 0; b < B; b++) {
        const PagedSeq s = paged_seq(w.seqs, b);
        CHECK(s.len >= 0 && s.len <= w.seqs.max_keys);
        CHECK(s.n >= 0 && s.q0 >= 0 && s.q0 + s.n <= w.seqs.total);
        const int32_t tiles = paged_row_tiles<ROWS>(w, s.n);
        CHECK(tiles == (s.n * w.G + ROWS - 1) / ROWS);
        const MaskSpec m = paged_mask(w.mask, s);
        int64_t units = 0;
        for (int32_t rt = 0; rt < tiles; rt++) {
            const PagedTile t = paged_tile<ROWS, BN>(w, s, rt);
            CHECK(t.units >= 1 && t.first >= 0);
            CHECK(t.hi < t.lo || (t.lo >= 0 && t.hi < s.len));
            units += t.units;
            for (int32_t r = rt * ROWS; r < (rt + 1) * ROWS && r < s.n * w.G; r += 3) {
                int lo, hi;
                row_key_bounds(m, r / w.G, lo, hi);
                for (int32_t key = 0; key < s.len; key++) {
                    const bool seen = key_visible(m, r / w.G, key);
                    CHECK(seen == (key >= lo && key <= hi));
                    CHECK(!seen || (key >= t.lo && key <= t.hi && key / BN >= t.first && key / BN < t.first + t.units));
                }
            }
        }
        CHECK((units == paged_head_units<ROWS, BN>(w, s)));
        total += units * w.Hkv;
    }
    const int32_t share = paged_share(w, (int32_t)total);
    CHECK(share >= w.min_units && (int64_t)share * w.n_wg >= total);
    for (int32_t t = 0; t < w.seqs.total; t++) {
        const int32_t b = paged_seq_of_row(w.seqs, t);
        CHECK(b >= -1 && b < B);
        if (!wild) {
            bool found = false;
            for (int32_t i = 0; i < B; i++) {
                const PagedSeq s = paged_seq(w.seqs, i);
                if (t >= s.q0 && t < s.q0 + s.n) {
                    CHECK(b == i);
                    found = true;
                }
            }
            CHECK(found || b == -1);
        }
    }
    CHECK(paged_rows_end(w.seqs) >= 0 && paged_rows_end(w.seqs) <= w.seqs.total);
}

int main() {
    for (long n = 0; n < 300; n++) {
        one<32, 32>(n);
        one<128, 64>(n);
        one<256, 64>(n);
    }
    // the largest lengths: no overflow (built with -fsanitize=signed-integer-overflow)
    for (int32_t window : {0, 1, (1 << 30) - 1}) {
        for (int32_t causal : {0, 1}) {
            const long n = -1;
            const int32_t big = 1 << 28;
            const int32_t lens[1] = {INT32_MAX};
            PagedWork w{};
            w.G = 4;
            w.Hkv = 1;
            w.seqs = PagedSeqs{lens, nullptr, 1, big, big, big};
            w.mask = PagedMask{causal, window};
            w.max_rows = INT32_MAX;
            const PagedSeq s = paged_seq(w.seqs, 0);
            const int32_t last = paged_row_tiles<256>(w, s.n) - 1;
            for (int32_t rt : {0, 1, last}) {
                const PagedTile t = paged_tile<256, 64>(w, s, rt);
                CHECK(t.units >= 1 && t.units <= big / 64 && t.first >= 0);
            }
        }
    }
    std::printf("ok %ld\n", checks);
    return 0;
}
