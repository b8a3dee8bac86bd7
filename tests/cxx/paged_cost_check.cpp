// Host check of paged_max_cost (rdnattention_amd/csrc/paged_rows.hpp): no lengths make
// a launch cost more, and calls that fit are not refused for rows of the other launch.
#include "paged_rows.hpp"

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>

using namespace rdna_amd;

static long checks = 0, n = 0;
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
#define CHECK(x)                                                      \
    do {                                                              \
        checks++;                                                     \
        if (!(x)) {                                                   \
            std::printf("line %d: %s (case %ld)\n", __LINE__, #x, n); \
            std::exit(1);                                             \
        }                                                             \
    } while (0)

template <int ROWS, int BN, int EXTRA>
static void one() {
    const int32_t B = pick(1, 8);
    std::vector<int32_t> lens(B), cu(B + 1, 0);
    PagedWork w{};
    w.G = pick(1, 9);
    w.Hkv = pick(1, 3);
    w.seqs.max_keys = pick(0, 2000);
    for (int32_t b = 0; b < B; b++) {
        cu[b + 1] = cu[b] + (rnd() % 3 ? pick(0, 40) : pick(0, 700));
        lens[b] = rnd() % 2 ? w.seqs.max_keys : pick(0, w.seqs.max_keys);
    }
    const bool ragged = rnd() % 4 != 0;
    w.seqs.rows = pick(1, 300);
    w.seqs.total = ragged ? cu[B] + pick(0, 3) : B * w.seqs.rows;
    w.seqs.cu = ragged ? cu.data() : nullptr;
    w.seqs.lens = lens.data();
    w.seqs.B = B;
    w.mask.causal = rnd() % 2;
    w.mask.window = rnd() % 2 ? 0 : pick(1, 200);
    w.min_rows = rnd() % 2 ? 0 : 32;
    w.max_rows = w.min_rows == 0 && rnd() % 2 ? 32 : INT32_MAX;
    int64_t cost = 0;
    for (int32_t b = 0; b < B; b++) {
        const PagedSeq s = paged_seq(w.seqs, b);
        cost += w.Hkv * ((int64_t)paged_head_units<ROWS, BN>(w, s) + EXTRA * paged_row_tiles<ROWS>(w, s.n));
    }
    CHECK((cost <= paged_max_cost<ROWS, BN, EXTRA>(w)));
    // a row's sequence, searched for from any sequence that is not behind it
    for (int32_t t = 0; ragged && t < w.seqs.total; t += 1 + t / 8) {
        const int32_t b = paged_seq_of_row(w.seqs, t);
        for (int32_t from = 0; from <= b; from++) {
            CHECK(paged_seq_of_row(w.seqs, t, from) == b);
        }
        CHECK(paged_seq_of_row(w.seqs, t, B) == -1);
    }
}

// A ragged call: rows of Hq / Hkv heads of B sequences over tables of `keys`.
static bool fits(int32_t rows, int32_t Hq, int32_t Hkv, int32_t B, int32_t keys) {
    static const int32_t none[2] = {0, 0};
    PagedWork w{};
    w.G = Hq / Hkv;
    w.Hkv = Hkv;
    w.seqs = PagedSeqs{none, none, B, 0, rows, keys};
    w.min_rows = 32;
    w.max_rows = INT32_MAX;
    const int64_t many = paged_max_cost<256, 64, 4>(w);
    w.min_rows = 0;
    w.max_rows = 32;
    return many <= INT32_MAX && paged_max_cost<32, 32, 0>(w) <= INT32_MAX;
}

int main() {
    for (n = 0; n < 20000; n++) {
        one<32, 32, 0>();
        one<128, 64, 4>();
        one<256, 64, 4>();
    }
    CHECK(fits(262144, 32, 8, 1, 262144)); // one long prompt
    CHECK(fits(65536, 32, 8, 1, 1 << 20)); // a chunk over a million keys
    CHECK(fits(32768, 64, 8, 1, 1 << 20));
    CHECK(fits(131072, 64, 8, 4, 262144));
    CHECK(fits(4096, 32, 8, 4096, 1 << 20));  // 4096 sequences with a million keys each
    CHECK(!fits(65600, 32, 8, 65536, 1 << 17)); // 2^31 key tiles of 32 keys
    CHECK(!fits(1 << 20, 64, 8, 1, 1 << 26));
    CHECK(!fits(1 << 28, 65535, 65535, 1 << 24, 1 << 28)); // past 63 bits
    std::printf("ok %ld\n", checks);
    return 0;
}
