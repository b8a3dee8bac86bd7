// Where the rows and keys of a paged call are: plain integer code, device
// functions when compiled as HIP, ordinary inline functions otherwise (host
// tests check them, tests/cxx/paged_rows_check.cpp).
//
// A call has B sequences.  Sequence b has `len` keys in its pages, the last n
// of them its newest rows: row i is key len - n + i.  The lengths, row ranges
// and page tables are device memory that the host does not see, so every value
// is bounded here and no access leaves a buffer, whatever they hold.
//
// The attention kernels deal a call's key tiles to their workers (workgroups): the
// rows (n tokens of G query heads each) of every (sequence, kv head) fall into row
// tiles of ROWS rows, and a row tile is an item of as many units as it sees key
// tiles of BN keys (one if none, for its zeros).  An item costs its units and
// EXTRA, what its begin and end take the time of, and worker w has the cost [w *
// share, (w + 1) * share) of the items in order (sequence, kv head, row tile).
// At most two of a worker's items are shared with others: the first and the last.
#pragma once

#include "fa_mask.hpp"

#include <cstdint>

namespace rdna_amd {

struct PagedSeqs {
    const int32_t* lens; // [B] keys in the cache
    const int32_t* cu;   // [B + 1] first row of each sequence, or null: `rows` each
    int32_t B;
    int32_t rows;
    int32_t total;    // rows of the query tensor
    int32_t max_keys; // keys that a row of the page table covers
    // The first `prefixes` of the B entries are prefixes: entry b has prefix_lens[b] keys and the
    // rows of sequences group[b] .. group[b + 1] - 1 of `members` (group null: of all of
    // them), and the entries behind them are the sequences themselves.
    int32_t prefixes = 0;
    int32_t members = 0;
    int32_t prefix_keys = 0; // keys that a row of the prefixes' page table covers
    const int32_t* prefix_lens = nullptr;
    const int32_t* group = nullptr;
};

struct PagedSeq {
    int32_t q0;  // first row in the query tensor
    int32_t n;   // rows
    int32_t len; // keys
};

RDNA_MASK_FN int32_t rows_clamp(int32_t x, int32_t lo, int32_t hi) {
    return mask_imin(mask_imax(x, lo), hi);
}

// Rows that belong to a sequence: [0, paged_rows_end).
RDNA_MASK_FN int32_t paged_rows_end(const PagedSeqs& s) {
    return s.cu != nullptr ? rows_clamp(s.cu[s.prefixes > 0 ? s.members : s.B], 0, s.total) : s.total;
}

RDNA_MASK_FN PagedSeq paged_seq(const PagedSeqs& s, int32_t b) {
    PagedSeq r;
    r.len = rows_clamp(s.lens[b], 0, s.max_keys);
    if (s.cu != nullptr) {
        r.q0 = rows_clamp(s.cu[b], 0, s.total);
        r.n = rows_clamp(s.cu[b + 1], r.q0, s.total) - r.q0;
    } else {
        r.q0 = b * s.rows;
        r.n = s.rows;
    }
    return r;
}

// Entry b of those that prefixes begin.
RDNA_MASK_FN PagedSeq paged_entry(const PagedSeqs& s, int32_t b) {
    if (b >= s.prefixes) {
        return paged_seq(s, b - s.prefixes);
    }
    PagedSeq r;
    r.len = rows_clamp(s.prefix_lens[b], 0, s.prefix_keys);
    const int32_t first = s.group != nullptr ? rows_clamp(s.group[b], 0, s.members) : 0;
    const int32_t end = s.group != nullptr ? rows_clamp(s.group[b + 1], first, s.members) : s.members;
    if (s.cu != nullptr) {
        r.q0 = rows_clamp(s.cu[first], 0, s.total);
        r.n = rows_clamp(s.cu[end], r.q0, s.total) - r.q0;
    } else {
        r.q0 = first * s.rows;
        r.n = (end - first) * s.rows;
    }
    return r;
}

// The sequence that row t of a ragged call belongs to, none before `from`: the first
// that ends behind it.  -1 for a row behind the last one.
RDNA_MASK_FN int32_t paged_seq_of_row(const PagedSeqs& s, int32_t t, int32_t from = 0) {
    if (s.cu == nullptr) {
        return t / s.rows;
    }
    while (from < s.B && s.cu[from + 1] <= t) {
        from++;
    }
    return from < s.B && s.cu[from] <= t ? from : -1;
}

// Visibility of a sequence's keys (see MaskSpec); a tree's prefix and drafts
// are one range here, its mask comes on top.
struct PagedMask {
    int32_t causal;
    int32_t window;
};

RDNA_MASK_FN MaskSpec paged_mask(const PagedMask& m, const PagedSeq& s) {
    return MaskSpec{s.len, s.len - s.n, m.causal, m.window};
}

// Rows lo .. hi (tokens times G and heads, none where hi < lo) of a sequence that see
// key `key`: neither falls as the key grows.
struct PagedKeyRows {
    int32_t lo, hi;
};
RDNA_MASK_FN PagedKeyRows paged_key_rows(const PagedMask& m, const PagedSeq& s, int32_t G, int32_t key) {
    // the first and the last token that sees it
    const int32_t at = key - (s.len - s.n);
    int32_t first = 0, last = s.n - 1;
    if (m.causal != 0) {
        first = at;
        if (m.window > 0) {
            last = at + m.window - 1;
        }
    } else if (m.window > 0) {
        first = at - (m.window >> 1);
        last = at + (m.window >> 1);
    }
    first = rows_clamp(first, 0, s.n);
    last = mask_imin(mask_imax(last, -1), s.n - 1);
    return key >= 0 && key < s.len ? PagedKeyRows{first * G, (last + 1) * G - 1} : PagedKeyRows{s.n * G, -1};
}

// Work of a call: sequences with more than min_rows and at most max_rows rows
// (tokens times G) are dealt to n_wg workers.
struct PagedWork {
    PagedSeqs seqs;
    PagedMask mask;
    int32_t Hkv, G;
    int32_t min_rows, max_rows;
    int32_t n_wg;
    int32_t min_units; // smallest share
};

// Row tiles of a sequence, 0 where another launch works on it.
template <int ROWS>
RDNA_MASK_FN int32_t paged_row_tiles(const PagedWork& w, int32_t n) {
    const int32_t rows = n * w.G;
    return rows > w.min_rows && rows <= w.max_rows ? (rows + ROWS - 1) / ROWS : 0;
}

// Key tiles of row tile rt: `units` from tile `first` on; nothing visible: units
// 1 and lo > hi.
struct PagedTile {
    int32_t lo, hi; // keys that some row sees
    int32_t first, units;
};

template <int ROWS, int BN>
RDNA_MASK_FN PagedTile paged_tile(const PagedWork& w, const PagedSeq& s, int32_t rt) {
    const int32_t i_lo = rt * ROWS / w.G;
    const int32_t i_hi = (mask_imin((rt + 1) * ROWS, s.n * w.G) - 1) / w.G;
    PagedTile t;
    visible_key_range(paged_mask(w.mask, s), i_lo, i_hi, t.lo, t.hi);
    if (t.hi < t.lo) {
        t.lo = 0;
        t.hi = -1;
        t.first = 0;
        t.units = 1;
    } else {
        t.first = t.lo / BN;
        t.units = t.hi / BN + 1 - t.first;
    }
    return t;
}

// Units of one kv head of a sequence, which has n row tiles.  (A caller that knows n to be small
// tells the compiler so: counted again here, it is a loop of 1.2 us at a kernel's begin.)
template <int ROWS, int BN>
RDNA_MASK_FN int32_t paged_head_units(const PagedWork& w, const PagedSeq& s, int32_t n) {
    int32_t u = 0;
    for (int32_t rt = 0; rt < n; rt++) {
        u += paged_tile<ROWS, BN>(w, s, rt).units;
    }
    return u;
}
template <int ROWS, int BN>
RDNA_MASK_FN int32_t paged_head_units(const PagedWork& w, const PagedSeq& s) {
    return paged_head_units<ROWS, BN>(w, s, paged_row_tiles<ROWS>(w, s.n));
}

// Items of a call: of a sequence and kv head its row tiles, whose units are key tiles.
template <int ROWS, int BN>
struct PagedRowItems {
    static RDNA_MASK_FN int32_t count(const PagedWork& w, const PagedSeq& s) {
        return paged_row_tiles<ROWS>(w, s.n);
    }
    static RDNA_MASK_FN PagedTile tile(const PagedWork& w, const PagedSeq& s, int32_t i) {
        return paged_tile<ROWS, BN>(w, s, i);
    }
    // of one kv head with n items
    static RDNA_MASK_FN int32_t units(const PagedWork& w, const PagedSeq& s, int32_t n) {
        return paged_head_units<ROWS, BN>(w, s, n);
    }
    // any of those whose rows see all keys
    static RDNA_MASK_FN PagedTile all(const PagedSeq& s) {
        return s.len > 0 ? PagedTile{0, s.len - 1, 0, (s.len + BN - 1) / BN} : PagedTile{0, -1, 0, 1};
    }
};

// ... or its blocks of BLOCK keys, whose units are the tiles of ROWS rows that see some key
// of theirs; lo .. hi are rows.
template <int BLOCK, int ROWS>
struct PagedKeyItems {
    static RDNA_MASK_FN int32_t count(const PagedWork& w, const PagedSeq& s) {
        const int32_t rows = s.n * w.G;
        return rows > w.min_rows && rows <= w.max_rows ? (s.len + BLOCK - 1) / BLOCK : 0;
    }
    static RDNA_MASK_FN PagedTile tile(const PagedWork& w, const PagedSeq& s, int32_t i) {
        const int32_t lo = paged_key_rows(w.mask, s, w.G, i * BLOCK).lo;
        const int32_t hi = paged_key_rows(w.mask, s, w.G, mask_imin((i + 1) * BLOCK, s.len) - 1).hi;
        return lo <= hi ? PagedTile{lo, hi, lo / ROWS, hi / ROWS + 1 - lo / ROWS} : PagedTile{0, -1, 0, 1};
    }
    static RDNA_MASK_FN int32_t units(const PagedWork& w, const PagedSeq& s, int32_t n) {
        int32_t u = 0;
        for (int32_t i = 0; i < n; i++) {
            u += tile(w, s, i).units;
        }
        return u;
    }
};

// Most that the items of a call may cost (see PagedShare), whatever the lengths: the
// sequences of a launch have more than min_rows and at most max_rows rows each, all of
// them `total` tokens.  Past 32 bits the walk cannot count it.
template <int ROWS, int BN, int EXTRA>
inline int64_t paged_max_cost(const PagedWork& w) {
    if (w.seqs.prefixes > 0) { // the prefixes' entries have all rows too
        PagedWork part = w;
        part.seqs.prefixes = 0;
        part.seqs.B = w.seqs.prefixes;
        part.seqs.max_keys = w.seqs.prefix_keys;
        const int64_t shared = paged_max_cost<ROWS, BN, EXTRA>(part);
        part.seqs.B = w.seqs.B - w.seqs.prefixes;
        part.seqs.max_keys = w.seqs.max_keys;
        const int64_t own = paged_max_cost<ROWS, BN, EXTRA>(part);
        return shared > INT32_MAX || own > INT32_MAX ? INT64_MAX : shared + own;
    }
    const int64_t rows = (int64_t)w.seqs.total * w.G;
    const int64_t B = w.seqs.B;
    const int64_t seqs = rows / ((int64_t)w.min_rows + 1) < B ? rows / ((int64_t)w.min_rows + 1) : B;
    const int64_t each = ((int64_t)w.max_rows - 1) / ROWS + 1;
    const int64_t tiles = rows / ROWS + seqs < seqs * each ? rows / ROWS + seqs : seqs * each;
    const int64_t heads = tiles * w.Hkv;
    return heads <= INT32_MAX ? heads * (w.seqs.max_keys / BN + 1 + EXTRA) : INT64_MAX;
}

// ... and those of blocks of keys.
template <int BLOCK, int ROWS, int EXTRA>
inline int64_t paged_max_key_cost(const PagedWork& w) {
    const int64_t rows = (int64_t)w.seqs.total * w.G;
    const int64_t B = w.seqs.B;
    const int64_t seqs = rows / ((int64_t)w.min_rows + 1) < B ? rows / ((int64_t)w.min_rows + 1) : B;
    const int64_t heads = (rows / ROWS + seqs * (2 + EXTRA)) * w.Hkv; // row tiles, whole or cut, and EXTRA
    return heads <= INT32_MAX ? heads * (w.seqs.max_keys / BLOCK + 1) : INT64_MAX;
}

// Cost of each worker's share of `total`.
RDNA_MASK_FN int32_t paged_share(const PagedWork& w, int32_t total) {
    return mask_imax(total / w.n_wg + (total % w.n_wg > 0 ? 1 : 0), w.min_units);
}

// Worker wg's share.  A caller that by mistake changes the lengths while a kernel
// runs gets wrong rows, but no access outside a buffer: whatever the items'
// units turn out to be, the parts lie inside their items, the slots and the last worker
// inside their arrays, and the walk ends.
template <int EXTRA>
struct PagedShare {
    int32_t n_wg, wg;
    int32_t left = 0;  // cost not yet taken
    int32_t at = 0;    // of the current item's cost, what earlier shares have
    int32_t start = 0; // of the call's cost, what lies before
    int32_t share = 1;

    RDNA_MASK_FN PagedShare(const PagedWork& w, int32_t worker) : n_wg(w.n_wg), wg(worker) {}

    RDNA_MASK_FN void deal(const PagedWork& w, int32_t total) {
        share = paged_share(w, total);
        start = (int64_t)wg * share < total ? wg * share : total;
        left = mask_imax(mask_imin(share, total - start), 0);
    }
    // The share begins in a sequence with `before` in front of it, each of whose
    // kv heads costs per_head > 0: that head.
    RDNA_MASK_FN int32_t enter(int32_t before, int32_t per_head, int32_t Hkv) {
        at = mask_imax(start - before, 0);
        const int32_t h = mask_imin(at / per_head, Hkv - 1);
        at -= h * per_head;
        return h;
    }
    // The current item is one of `units`: nothing is left if none of them is in the
    // share.
    RDNA_MASK_FN void item(int32_t units) {
        at = rows_clamp(at, 0, units + EXTRA - 1);
        if (at + left <= EXTRA) {
            left = 0;
        }
    }
    RDNA_MASK_FN bool more() const {
        return left > 0;
    }
    RDNA_MASK_FN int32_t cost(int32_t units) const {
        return mask_imin(left, units + EXTRA - at);
    }
    // The part of the item in this share: units [begin, begin + count).
    RDNA_MASK_FN int32_t begin() const {
        return mask_imax(at - EXTRA, 0);
    }
    RDNA_MASK_FN int32_t count(int32_t units) const {
        return at + cost(units) - EXTRA - begin();
    }
    RDNA_MASK_FN bool whole(int32_t units) const {
        return begin() == 0 && at + cost(units) == units + EXTRA;
    }
    // Slot of a part that is not the whole item, and, of the first part, the last
    // worker.
    RDNA_MASK_FN int32_t slot() const {
        return begin() == 0 ? n_wg + wg : wg;
    }
    RDNA_MASK_FN int32_t last_wg(int32_t units) const {
        const uint32_t end = (uint32_t)(start - at) + (uint32_t)(units + EXTRA - 1);
        return mask_imax((int32_t)(end / (uint32_t)share < (uint32_t)n_wg ? end / (uint32_t)share : n_wg - 1), wg);
    }
    // On to the next item, which is still to be given to item().
    RDNA_MASK_FN void take(int32_t units) {
        const int32_t n = cost(units);
        left -= n;
        start += n;
        at = 0;
    }
};

} // namespace rdna_amd
