// Host check of PagedShare (rdnattention_amd/csrc/paged_rows.hpp): the shares of a
// call have every unit of every item exactly once, the records lead the merge to
// all parts of an item and to nothing else, and items whose units change while the
// workers walk over them still end every walk with every index in its array.
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

struct Seq {
    std::vector<int32_t> units; // of the row tiles of one kv head
};

template <int EXTRA>
static void dealt() {
    const int32_t Hkv = pick(1, 4), B = pick(1, 5);
    std::vector<Seq> seqs(B);
    int32_t total = 0;
    std::vector<int32_t> per_head(B, 0), first(B + 1, 0); // items before a sequence
    for (int32_t b = 0; b < B; b++) {
        for (int32_t i = pick(0, 6); i > 0; i--) {
            seqs[b].units.push_back(rnd() % 4 == 0 ? 1 : pick(1, 40));
            per_head[b] += seqs[b].units.back() + EXTRA;
        }
        total += per_head[b] * Hkv;
        first[b + 1] = first[b] + Hkv * (int32_t)seqs[b].units.size();
    }
    PagedWork w{};
    w.n_wg = pick(1, 70);
    w.min_units = pick(1, 8);

    const int32_t items = first[B];
    std::vector<std::vector<int>> taken(items);
    for (int32_t b = 0, k = 0; b < B; b++) {
        for (int32_t h = 0; h < Hkv; h++) {
            for (int32_t u : seqs[b].units) {
                taken[k++].assign(u, 0);
            }
        }
    }
    std::vector<int32_t> slot_item(2 * w.n_wg, -1), rec_item(w.n_wg, -1), rec_last(w.n_wg, -1), parts(items, 0),
        wholes(items, 0);
    for (int32_t wg = 0; wg < w.n_wg; wg++) {
        PagedShare<EXTRA> s(w, wg);
        s.deal(w, total);
        if (!s.more()) {
            continue;
        }
        // the sequence, kv head and row tile that the share begins in
        int32_t b = 0, before = 0;
        while (before + per_head[b] * Hkv <= s.start) {
            before += per_head[b++] * Hkv;
        }
        int32_t h = s.enter(before, per_head[b], Hkv);
        int32_t rt = 0;
        while (s.at >= seqs[b].units[rt] + EXTRA) {
            s.at -= seqs[b].units[rt++] + EXTRA;
        }
        s.item(seqs[b].units[rt]);
        while (s.more()) {
            const int32_t tiles = (int32_t)seqs[b].units.size(), units = seqs[b].units[rt];
            const int32_t k = first[b] + h * tiles + rt;
            CHECK(s.begin() >= 0 && s.count(units) >= 1 && s.begin() + s.count(units) <= units);
            for (int32_t u = s.begin(); u < s.begin() + s.count(units); u++) {
                taken[k][u]++;
            }
            if (s.whole(units)) {
                wholes[k]++;
            } else {
                CHECK(slot_item[s.slot()] == -1);
                slot_item[s.slot()] = k;
                parts[k]++;
                if (s.begin() == 0) {
                    CHECK(rec_item[wg] == -1);
                    rec_item[wg] = k;
                    rec_last[wg] = s.last_wg(units);
                }
            }
            s.take(units);
            if (!s.more()) {
                break;
            }
            if (++rt == tiles) {
                rt = 0;
                if (++h == Hkv) {
                    h = 0;
                    do {
                        b++;
                        CHECK(b < B);
                    } while (seqs[b].units.empty());
                }
            }
            s.item(seqs[b].units[rt]);
        }
    }
    for (int32_t k = 0; k < items; k++) {
        for (int c : taken[k]) {
            CHECK(c == 1);
        }
        CHECK(wholes[k] + (parts[k] > 0) == 1);
    }
    std::vector<int32_t> merged(items, 0);
    for (int32_t wg = 0; wg < w.n_wg; wg++) {
        if (rec_item[wg] >= 0) {
            CHECK(rec_last[wg] > wg && rec_last[wg] < w.n_wg);
            CHECK(slot_item[w.n_wg + wg] == rec_item[wg]);
            for (int32_t i = wg + 1; i <= rec_last[wg]; i++) {
                CHECK(slot_item[i] == rec_item[wg]);
            }
            merged[rec_item[wg]] += rec_last[wg] - wg + 1;
        }
    }
    for (int32_t k = 0; k < items; k++) {
        CHECK(merged[k] == parts[k]);
    }
}

// Units that are others at every look, sums that have wrapped.
template <int EXTRA>
static void changing() {
    PagedWork w{};
    w.n_wg = pick(1, 70);
    w.min_units = pick(1, 8);
    const int32_t total = rnd() % 8 == 0 ? (int32_t)rnd() : rnd() % 4 == 0 ? INT32_MAX - pick(0, 99) : pick(0, 5000);
    const auto any_units = [] { return rnd() % 3 == 0 ? 1 << 22 : pick(1, 300); };
    for (int32_t wg = 0; wg < w.n_wg; wg++) {
        PagedShare<EXTRA> s(w, wg);
        s.deal(w, total);
        CHECK(s.left >= 0 && s.left <= s.share);
        if (!s.more()) {
            continue;
        }
        const int32_t Hkv = pick(1, 9);
        const int32_t h = s.enter(rnd() % 2 ? (int32_t)(rnd() >> 1) : s.start, pick(1, 4000), Hkv);
        CHECK(h >= 0 && h < Hkv);
        if (rnd() % 3 == 0) {
            s.at = (int32_t)rnd();
        }
        int32_t units = any_units();
        s.item(units);
        for (int32_t step = 0; s.more(); step++) {
            CHECK(step < 200000 && s.cost(units) >= 1);
            CHECK(s.begin() >= 0 && s.count(units) >= 1 && s.begin() + s.count(units) <= units);
            CHECK(s.slot() >= 0 && s.slot() < 2 * w.n_wg);
            CHECK(s.last_wg(units) >= wg && s.last_wg(units) < w.n_wg);
            s.take(units);
            units = any_units();
            s.item(units);
        }
    }
}

int main() {
    for (n = 0; n < 3000; n++) {
        dealt<0>();
        dealt<4>();
        if (n < 300) {
            changing<0>();
            changing<4>();
        }
    }
    std::printf("ok %ld\n", checks);
    return 0;
}
