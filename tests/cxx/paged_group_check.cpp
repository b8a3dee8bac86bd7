// paged_entry of prefixes, which stand for groups of sequences, and of the sequences behind them: the rows of the group where
// the arrays make sense, rows inside the tensors whatever they hold.
#include "paged_rows.hpp"

#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

using namespace rdna_amd;

#define CHECK(c)                                                                                                       \
    do {                                                                                                               \
        if (!(c)) {                                                                                                    \
            std::printf("line %d: %s\n", __LINE__, #c);                                                                \
            return 1;                                                                                                  \
        }                                                                                                              \
    } while (0)

int main() {
    std::mt19937 rng(1);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    long checked = 0;
    for (int it = 0; it < 200000; it++) {
        const int seqs = pick(1, 12), groups = pick(1, 6);
        const bool ragged = pick(0, 1) != 0, sane = pick(0, 1) != 0;
        const int rows = pick(1, 5);
        std::vector<int> cu(seqs + 1), group(groups + 1), lens(groups);
        int at = 0;
        for (int b = 0; b <= seqs; b++) {
            cu[b] = ragged ? at : b * rows;
            at += pick(0, 7);
        }
        const int total = ragged ? cu[seqs] + pick(0, 4) : seqs * rows;
        for (int g = 1; g <= groups; g++) {
            group[g] = g == groups ? seqs : pick(group[g - 1], seqs);
        }
        for (int& n : lens) {
            n = sane ? pick(0, 100) : pick(0, 1) != 0 ? INT_MAX : INT_MIN;
        }
        if (!sane) {
            const int odd[] = {INT_MIN, -1, 0, 3, seqs, total, INT_MAX};
            for (int& x : cu) {
                x = odd[pick(0, 6)];
            }
            for (int& x : group) {
                x = odd[pick(0, 6)];
            }
        }
        std::vector<int> own(seqs);
        for (int& n : own) {
            n = sane ? pick(0, 60) : pick(0, 1) != 0 ? INT_MAX : INT_MIN;
        }
        PagedSeqs s{own.data(), ragged ? cu.data() : nullptr, groups + seqs, rows, total, 50};
        s.prefixes = groups;
        s.members = seqs;
        s.prefix_keys = 80;
        s.prefix_lens = lens.data();
        s.group = groups == 1 && pick(0, 1) != 0 ? nullptr : group.data();
        int next = 0;
        for (int g = 0; g < groups; g++) {
            const PagedSeq r = paged_entry(s, g);
            CHECK(r.q0 >= 0 && r.n >= 0 && r.n <= total && r.q0 <= total - r.n);
            CHECK(r.len >= 0 && r.len <= 80);
            if (sane) {
                CHECK(r.q0 == next && r.len == (lens[g] < 80 ? lens[g] : 80));
                next = r.q0 + r.n;
            }
            checked++;
        }
        for (int b = 0; b < seqs; b++) {
            const PagedSeq r = paged_entry(s, groups + b);
            CHECK(r.q0 >= 0 && r.n >= 0 && r.n <= total && r.q0 <= total - r.n && r.len >= 0 && r.len <= 50);
            CHECK(!sane || (r.q0 == cu[b] && r.n == cu[b + 1] - cu[b] && r.len == (own[b] < 50 ? own[b] : 50)));
            checked++;
        }
        CHECK(!sane || paged_rows_end(s) == (ragged ? cu[seqs] : total));
        CHECK(!sane || next == (ragged ? cu[seqs] : total));
    }
    std::printf("ok %ld\n", checked);
    return 0;
}
