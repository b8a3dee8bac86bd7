// paged_key_rows against the rule of visibility, row by row, and at the largest values.
#include "paged_rows.hpp"

#include <cstdio>
#include <random>

using namespace rdna_amd;

#define CHECK(c)                                                                                                       \
    do {                                                                                                               \
        if (!(c)) {                                                                                                    \
            std::printf("line %d: %s\n", __LINE__, #c);                                                                \
            return 1;                                                                                                  \
        }                                                                                                              \
    } while (0)

int main() {
    std::mt19937 rng(2);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    long checked = 0;
    for (int it = 0; it < 100000; it++) {
        const PagedSeq s{0, pick(1, 12), pick(0, 20)};
        const PagedMask m{pick(0, 1), pick(0, 2) == 0 ? 0 : pick(1, 9)};
        const int G = pick(1, 5);
        int lo = 0, hi = -1;
        for (int key = -1; key < s.len + 2; key++) {
            const PagedKeyRows r = paged_key_rows(m, s, G, key);
            for (int row = 0; row < s.n * G; row++) {
                const bool sees = key >= 0 && key_visible(paged_mask(m, s), row / G, key);
                CHECK(sees == (row >= r.lo && row <= r.hi));
                checked++;
            }
            if (key >= 0 && key < s.len) { // neither falls
                CHECK(r.lo >= lo && r.hi >= hi);
                lo = r.lo;
                hi = r.hi;
            }
        }
    }
    const int big = 1 << 28;
    for (int n : {1, big}) {
        for (int len : {0, 1, big}) {
            for (int causal : {0, 1}) {
                for (int window : {0, 1, (1 << 30) - 1}) {
                    for (int key : {0, 1, big - 1, big + 127}) {
                        const int G = n == big ? 4 : 65535;
                        const PagedKeyRows r = paged_key_rows(PagedMask{causal, window}, PagedSeq{0, n, len}, G, key);
                        CHECK(r.lo >= 0 && r.lo <= n * G && r.hi >= -1 && r.hi < n * G);
                        checked++;
                    }
                }
            }
        }
    }
    std::printf("ok %ld\n", checked);
    return 0;
}
