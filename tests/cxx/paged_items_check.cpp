// Host check of what the paged walks deal beside plain row tiles (rdnattention_amd/csrc/
// paged_rows.hpp): blocks of keys, and entries of prefixes.  Every row that sees a key of an item
// is in its units, prefixes' items are all alike, no lengths make a launch cost more than its bound,
// and the shares have every unit once.
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

struct Call {
    std::vector<int32_t> lens, cu, prefix_lens, group;
    PagedWork w{};
};

static void make(Call& c, bool prefixes) {
    const int32_t B = pick(1, 7);
    c.lens.resize(B);
    c.cu.assign(B + 1, 0);
    PagedWork& w = c.w;
    w.G = pick(1, 9);
    w.Hkv = pick(1, 3);
    w.seqs.max_keys = pick(0, 700);
    for (int32_t b = 0; b < B; b++) {
        c.cu[b + 1] = c.cu[b] + (rnd() % 3 ? pick(0, 40) : pick(0, 200));
        c.lens[b] = rnd() % 2 ? w.seqs.max_keys : pick(-3, w.seqs.max_keys + 3);
    }
    const bool ragged = rnd() % 4 != 0;
    w.seqs.rows = pick(1, 150);
    w.seqs.total = ragged ? c.cu[B] + pick(0, 3) : B * w.seqs.rows;
    w.seqs.cu = ragged ? c.cu.data() : nullptr;
    w.seqs.lens = c.lens.data();
    w.seqs.B = B;
    w.mask.causal = rnd() % 2;
    w.mask.window = rnd() % 2 || prefixes ? 0 : pick(1, 200);
    w.min_rows = rnd() % 2 ? 0 : pick(32, 128);
    w.max_rows = w.min_rows == 0 && rnd() % 2 ? 128 : INT32_MAX;
    w.n_wg = pick(1, 64);
    w.min_units = pick(1, 48);
    if (prefixes) {
        const int32_t P = pick(1, 4);
        c.prefix_lens.resize(P);
        c.group.assign(P + 1, 0);
        for (int32_t i = 0; i < P; i++) {
            c.prefix_lens[i] = pick(-2, 400);
            c.group[i + 1] = i + 1 == P ? B : pick(c.group[i], B);
        }
        w.min_rows = 0;
        w.max_rows = INT32_MAX;
        w.seqs.prefixes = P;
        w.seqs.members = B;
        w.seqs.prefix_keys = pick(0, 350);
        w.seqs.prefix_lens = c.prefix_lens.data();
        w.seqs.group = P == 1 && rnd() % 2 ? nullptr : c.group.data();
        w.seqs.B = P + (rnd() % 2 ? B : 0);
    }
}

// The units of a launch's items, entry after entry, dealt: each once, and what a worker has of an
// item at its share's ends only.
template <int EXTRA>
static void deal(PagedWork w, const std::vector<std::vector<int32_t>>& entries) {
    int64_t total = 0;
    std::vector<int32_t> per_head;
    for (const auto& units : entries) {
        int32_t u = 0;
        for (int32_t x : units) {
            u += x + EXTRA;
        }
        per_head.push_back(u);
        total += (int64_t)u * w.Hkv;
    }
    CHECK(total <= INT32_MAX);
    int64_t taken = 0, wanted = 0;
    for (const auto& units : entries) {
        for (int32_t x : units) {
            wanted += (int64_t)x * w.Hkv;
        }
    }
    // (item, units done of it): the workers have them in order
    size_t b_done = 0, i_done = 0;
    int32_t h_done = 0, u_done = 0;
    const auto skip_empty = [&] {
        while (b_done < entries.size() && entries[b_done].empty()) {
            b_done++;
        }
    };
    skip_empty();
    for (int32_t wg = 0; wg < w.n_wg; wg++) {
        PagedShare<EXTRA> s(w, wg);
        s.deal(w, (int32_t)total);
        if (!s.more()) {
            continue;
        }
        size_t b = 0;
        int32_t before = 0;
        while (before + per_head[b] * w.Hkv <= s.start) {
            before += per_head[b++] * w.Hkv;
        }
        int32_t h = s.enter(before, per_head[b], w.Hkv);
        size_t i = 0;
        while (s.at >= entries[b][i] + EXTRA) {
            s.at -= entries[b][i++] + EXTRA;
        }
        s.item(entries[b][i]);
        bool first = true;
        while (s.more()) {
            const int32_t units = entries[b][i];
            CHECK(b == b_done && h == h_done && i == i_done && s.begin() == u_done && s.count(units) >= 1);
            CHECK(first || s.begin() == 0);
            first = false;
            taken += s.count(units);
            u_done += s.count(units);
            CHECK(u_done <= units);
            CHECK(s.whole(units) == (s.begin() == 0 && s.count(units) == units));
            if (u_done == units) {
                u_done = 0;
                if (++i_done == entries[b].size()) {
                    i_done = 0;
                    if (++h_done == w.Hkv) {
                        h_done = 0;
                        b_done++;
                        skip_empty();
                    }
                }
            }
            s.take(units);
            if (!s.more()) {
                break;
            }
            if (++i == entries[b].size()) {
                i = 0;
                if (++h == w.Hkv) {
                    h = 0;
                    do {
                        b++;
                        CHECK(b < entries.size());
                    } while (entries[b].empty());
                }
            }
            s.item(entries[b][i]);
        }
    }
    CHECK(taken == wanted && b_done == entries.size());
}

template <int BLOCK, int ROWS, int EXTRA>
static void blocks_of_keys() {
    using Items = PagedKeyItems<BLOCK, ROWS>;
    Call c;
    make(c, false);
    const PagedWork& w = c.w;
    int64_t cost = 0;
    std::vector<std::vector<int32_t>> entries;
    for (int32_t b = 0; b < w.seqs.B; b++) {
        const PagedSeq s = paged_seq(w.seqs, b);
        const int32_t items = Items::count(w, s), rows = s.n * w.G;
        CHECK(items == (rows > w.min_rows && rows <= w.max_rows ? (s.len + BLOCK - 1) / BLOCK : 0));
        std::vector<int32_t> units;
        for (int32_t i = 0; i < items; i++) {
            const PagedTile t = Items::tile(w, s, i);
            CHECK(t.units >= 1 && t.first >= 0);
            CHECK(t.hi < t.lo ? t.units == 1 : t.lo >= 0 && t.hi < rows && t.first == t.lo / ROWS &&
                                                   t.first + t.units == t.hi / ROWS + 1);
            for (int32_t r = 0; r < rows; r += 1 + w.G / 2) {
                bool sees = false;
                for (int32_t key = i * BLOCK; key < (i + 1) * BLOCK && key < s.len; key++) {
                    sees |= key_visible(paged_mask(w.mask, s), r / w.G, key);
                }
                CHECK(!sees || (r >= t.lo && r <= t.hi));
            }
            units.push_back(t.units);
            cost += (int64_t)w.Hkv * (t.units + EXTRA);
        }
        int32_t sum = 0;
        for (int32_t u : units) {
            sum += u;
        }
        CHECK(sum == Items::units(w, s, items));
        entries.push_back(units);
    }
    CHECK((cost <= paged_max_key_cost<BLOCK, ROWS, EXTRA>(w)));
    deal<EXTRA>(w, entries);
}

template <int ROWS, int BN, int EXTRA>
static void entries_of_prefixes() {
    using Items = PagedRowItems<ROWS, BN>;
    Call c;
    make(c, true);
    const PagedWork& w = c.w;
    PagedWork unmasked = w;
    unmasked.mask = PagedMask{0, 0};
    int64_t cost = 0;
    std::vector<std::vector<int32_t>> entries;
    for (int32_t b = 0; b < w.seqs.B; b++) {
        const PagedSeq s = paged_entry(w.seqs, b);
        const bool prefix = b < w.seqs.prefixes;
        const int32_t items = Items::count(w, s);
        std::vector<int32_t> units;
        for (int32_t i = 0; i < items; i++) {
            const PagedTile t = Items::tile(prefix ? unmasked : w, s, i);
            if (prefix) {
                const PagedTile all = Items::all(s);
                CHECK(t.lo == all.lo && t.hi == all.hi && t.first == all.first && t.units == all.units);
                CHECK(s.len <= 0 || (t.lo == 0 && t.hi == s.len - 1));
            }
            units.push_back(t.units);
            cost += (int64_t)w.Hkv * (t.units + EXTRA);
        }
        int32_t sum = 0;
        for (int32_t u : units) {
            sum += u;
        }
        CHECK(sum == Items::units(prefix ? unmasked : w, s, items));
        entries.push_back(units);
    }
    CHECK((cost <= paged_max_cost<ROWS, BN, EXTRA>(w)));
    deal<EXTRA>(w, entries);
}

int main() {
    for (n = 0; n < 6000; n++) {
        blocks_of_keys<64, 32, 24>();
        blocks_of_keys<96, 32, 24>();
        blocks_of_keys<128, 32, 24>();
        entries_of_prefixes<32, 32, 24>();
        entries_of_prefixes<256, 64, 4>();
        entries_of_prefixes<128, 64, 4>();
    }
    std::printf("ok %ld\n", checks);
    return 0;
}
