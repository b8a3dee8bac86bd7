// Body of the paged_tiles kernels (paged_tiles.hpp), included into each of them.  In
// scope: T, D, I8, JOIN (rows whose keys are in two parts, or whose log-sum-exp is
// asked for), join and the parameters p.
    using C = TileCfg<D, I8>;
    using V8 = typename PagedVec<T>::v8;
    using V4 = typename PagedVec<T>::v4;
    using P = std::conditional_t<I8, _Float16, T>; // weights and values, see paged_stream
    using P8 = typename PagedVec<P>::v8;
    // the K slots, the V slots, the waves' table entries (int8: the scales), the waves' Q
    __shared__ __attribute__((aligned(16))) char dsm[C::LDS_BYTES];

    const int tid = threadIdx.x;
    const int wave = uniform(tid >> 6);
    const int lane = tid & 63;
    const int l32 = lane & 31;
    const int g = lane >> 5;
    const bool second = C::SPLIT && wave >= 4; // stages keys
    constexpr int V_SLOTS = 2 * C::TILE_BYTES;
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(dsm);
    constexpr int TABS = 2 * V_SLOTS;
    constexpr int QS = TABS + C::TAB_BYTES;
    const uint32_t page_mask = (1u << p.c.lps) - 1u;

    // LDS addresses of the MFMA operands in slot 0: K by s (+ 32 rows: kt), V by (dt, hh)
    // (+ 16 rows: u; the swizzle has a period of 16 rows).  Where registers are short they are
    // made for every tile, from an opaque copy of the lane so that they are not kept.
    auto addresses = [&](int ln, uint32_t (&ka)[C::KA], uint32_t (&va)[2 * C::VA]) RDNA_INLINE {
        const int row = ln & 31, j16 = ln & 15;
#pragma unroll
        for (int s = 0; s < C::KA; s++) {
            ka[s] = lds0 + row * C::RB + (((2 * s + (ln >> 5)) ^ paged_swz<D>(row)) << 4);
        }
#pragma unroll
        for (int x = 0; x < 2 * C::VA; x++) {
            const int r = 8 * (x & 1) + 4 * (ln >> 5) + (j16 >> 2);
            const int d = 32 * (x >> 1) + 16 * ((ln >> 4) & 1) + 4 * (j16 & 3);
            va[x] = lds0 + V_SLOTS + r * C::RB + (((d >> 3) ^ paged_swz<D>(r)) << 4) + ((d & 7) << 1);
        }
    };
    uint32_t ka0[C::KA], va0[2 * C::VA];
    if constexpr (C::KEEP) {
        addresses(lane, ka0, va0);
    }

    if (p.zero_tail != 0) {
        zero_tail_rows<D>(p, join.lse);
    }
    PagedRecord rec = {};
    // row tiles of one head, which read the same keys, through one L2
    PagedWalk<C::ROWS, kBN, true, kItemCost, JOIN> walk(p.work, by_xcd(blockIdx.x, p.work.n_wg));

    const int log_n = max(0, 6 - p.c.lps); // table entries of a tile
    const int log_b = 6 - log_n;           // tiles of a batch of 64
    auto tab_rsrc = [&](int b) RDNA_INLINE {
        i32x4_t r = make_rsrc_v(p.c.table + b * p.c.table_s, (uint32_t)p.c.width * 4u);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            r[e] = uniform(r[e]);
        }
        return r;
    };
    // entries of a batch of the item in half `odd` of the wave's, from key tile t0 on
    auto issue_tab = [&](i32x4_t rsrc, int odd, int t0, int batch) RDNA_INLINE {
        const int t = (batch << log_b) + (lane >> log_n);
        const int key = (t0 + t) * kBN + ((lane & ((1 << log_n) - 1)) << p.c.lps);
        dma_load4(rsrc, (uint32_t)(key >> p.c.lps) * 4u,
                  (uint32_t)uniform((int)lds0 + TABS + 2048 * wave + 1024 * odd + 256 * (batch & 3)));
    };
    // An item's row `col` of the wave's rows, the first one for those behind the last.
    auto token_head = [&](const auto& w, int& tok, int& head) RDNA_INLINE {
        const int r0 = uniform(w.rt) * C::ROWS, col = 32 * wave + l32;
        const bool valid = r0 + col < w.seq.n * p.work.G;
        const int r = valid ? r0 + col : r0;
        tok = r / p.work.G;
        head = uniform(w.h) * p.work.G + r - tok * p.work.G;
        return valid;
    };
    auto q_row = [&](const auto& w, int tok, int head) RDNA_INLINE {
        return p.q + (int64_t)(w.seq.q0 + tok) * p.q_st + head * p.q_sh;
    };
    // What an item needs first: Q (copy n's byte 16 lane is chunk 64 n + lane of the
    // wave's 32 rows; the lane of row r has its address) and two batches of entries.
    auto prefetch = [&](const auto& w, int odd) RDNA_INLINE {
        if constexpr (!I8) {
            const i32x4_t rsrc = tab_rsrc(w.b);
            const int t0 = uniform(w.tile.first + w.begin());
            issue_tab(rsrc, odd, t0, 0);
            issue_tab(rsrc, odd, t0, 1);
        }
        if constexpr (C::Q_LDS) {
            int tok, head;
            token_head(w, tok, head);
            const uint64_t mine = reinterpret_cast<uint64_t>(q_row(w, tok, head));
            const uint32_t lo = (uint32_t)mine, hi = (uint32_t)(mine >> 32);
            int ln = lane;
            asm volatile("" : "+v"(ln));
#pragma unroll
            for (int n = 0; n < C::NS; n++) {
                const int c = 64 * n + ln;
                const int r = c / C::KCH;
                const uint64_t row = (uint64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(4 * r, (int)hi) << 32 |
                                     (uint32_t)__builtin_amdgcn_ds_bpermute(4 * r, (int)lo);
                dma_gather16(row + (uint32_t)((c - r * C::KCH) ^ paged_swz<D>(r)) * 16u,
                             (uint32_t)uniform((int)lds0 + QS + wave * C::Q_BYTES + 1024 * n));
            }
        }
    };

    int odd = 0;
    if (walk.more()) {
        prefetch(walk, odd);
    }
    while (walk.more()) {
        const PagedSeq seq = walk.seq;
        const PagedTile item = walk.tile;
        const bool whole = walk.whole();
        const int h = uniform(walk.h);
        const int G = p.work.G;
        const int r0 = uniform(walk.rt) * C::ROWS;
        const int n_rows = min(C::ROWS, seq.n * G - r0);
        const int wr0 = 32 * wave; // of the item
        const int col = wr0 + l32;
        const bool active = wr0 < n_rows; // the wave
        int tok, head;
        const bool col_valid = token_head(walk, tok, head);
        const MaskSpec mask = paged_mask(p.work.mask, seq);
        int row_lo, row_hi;
        row_key_bounds(mask, tok, row_lo, row_hi);
        if (!col_valid) {
            row_lo = 1;
            row_hi = 0;
        }
        const int prefix = seq.len - seq.n;
        const uint8_t* tree_row = nullptr;
        int tree_n = 0;
        if (p.tree != nullptr) {
            tree_n = tok < p.tree_n ? min(p.tree_n, seq.n) : 0;
            tree_row = p.tree + walk.b * p.tree_sb + (tok < p.tree_n ? tok : 0) * p.tree_sr;
        }
        // the wave's classes of key tiles (see TileClasses)
        const TileClasses cls =
            active ? tile_classes<kBN>(mask, uniform((r0 + wr0) / G), uniform((r0 + min(wr0 + 32, n_rows) - 1) / G))
                   : TileClasses{1, 0, 1, 0};
        const int tree_from = p.tree != nullptr ? prefix : INT32_MAX; // keys from here on are under the tree's mask

        const int t0 = uniform(item.first + walk.begin());
        const int nt = uniform(item.hi >= item.lo ? walk.count() : 0);
        const char* const kbase = p.c.k + h * p.c.k_sh;
        const char* const vbase = p.c.v + h * p.c.v_sh;
        const uint32_t* const tab = reinterpret_cast<const uint32_t*>(dsm + TABS) + 512 * wave + 256 * odd;

        // ---- staging of 16-bit pages.  Copy d of a tile writes its LDS bytes 1024 d + 16
        // lane; wave w has copies w % 4, w % 4 + 4, ...
        // Copy d of keys or values (base, page and token strides) of tile t: each lane
        // finds its row.
        auto copy = [&](int t, int d, uint32_t lds, const char* base, int64_t sp, int64_t st) RDNA_INLINE {
            const int key0 = (t0 + t) * kBN;
            int ln = lane;
            asm volatile("" : "+v"(ln)); // no constants of every copy in registers
            const int n = 64 * d + ln;
            const int r = n / C::KCH;
            const bool seen = key0 + r >= item.lo && key0 + r <= item.hi;
            const uint32_t pg = tab[64 * ((t >> log_b) & 3) + ((t & ((1 << log_b) - 1)) << log_n) + (r >> p.c.lps)];
            const uint64_t pe = pg < (uint32_t)p.c.pages ? pg : 0u;
            const uint64_t off = (uint32_t)(key0 + r) & page_mask;
            const uint64_t row = reinterpret_cast<uint64_t>(base) + pe * (uint64_t)sp + off * (uint64_t)st;
            dma_gather16((seen ? row : reinterpret_cast<uint64_t>(kPagedZeroRow)) +
                             (uint32_t)((n - r * C::KCH) ^ paged_swz<D>(r)) * 16u,
                         lds);
        };
        // Where each copy's rows lie in one page, and every key of the tile is seen by a row
        // of the item: lane x finds the first row of copy x, and a copy's address is one
        // scalar and the lane's constant part.  (Finding them in turn took 20 us of the
        // 770 of B4 Hq32 Hkv8 S4096 D128 causal.)
        constexpr int CROWS = 1024 / C::RB;
        const bool one_page = 1024 % C::RB == 0 && (1 << p.c.lps) >= CROWS && (uint64_t)p.c.k_sp < (1ull << 32) &&
                              (uint64_t)p.c.v_sp < (1ull << 32) && p.c.k_st < (1 << 26) && p.c.v_st < (1 << 26);
        auto stage_copies = [&](bool values, int t) RDNA_INLINE {
            if (t >= nt) {
                return;
            }
            if ((C::SPLIT || !values) && t > 0 && (t & ((1 << log_b) - 1)) == 0) {
                issue_tab(tab_rsrc(walk.b), odd, t0, (t >> log_b) + 1); // over entries of three batches ago
            }
            const char* const base = values ? vbase : kbase;
            const int64_t sp = values ? p.c.v_sp : p.c.k_sp;
            const int64_t st = values ? p.c.v_st : p.c.k_st;
            const uint32_t slot = lds0 + (values ? V_SLOTS : 0) + (uint32_t)(t & 1) * C::TILE_BYTES;
            const int key0 = (t0 + t) * kBN;
            if (one_page && key0 >= item.lo && key0 + kBN - 1 <= item.hi) {
                int ln = lane;
                asm volatile("" : "+v"(ln));
                const int r = CROWS * ((wave & 3) + 4 * ln) & (kBN - 1);
                const uint32_t pg = tab[64 * ((t >> log_b) & 3) + ((t & ((1 << log_b) - 1)) << log_n) + (r >> p.c.lps)];
                const uint32_t pe = pg < (uint32_t)p.c.pages ? pg : 0u;
                const uint32_t off = (uint32_t)(key0 + r) & page_mask;
                const uint64_t row = reinterpret_cast<uint64_t>(base) + (uint64_t)pe * (uint32_t)sp +
                                     (uint64_t)off * (uint32_t)st;
                const int crow = lane / C::KCH;
#pragma unroll
                for (int x = 0; x < C::PER; x++) {
                    const int d = (wave & 3) + 4 * x;
                    dma_uniform16(readlane64(row, x),
                                  (uint32_t)crow * (uint32_t)st +
                                      (uint32_t)((lane % C::KCH) ^ paged_swz<D>(CROWS * d + crow)) * 16u,
                                  slot + 1024 * d);
                }
            } else {
#pragma unroll
                for (int x = 0; x < C::PER; x++) {
                    const int d = (wave & 3) + 4 * x;
                    copy(t, d, slot + 1024 * d, base, sp, st);
                }
            }
        };
        // int8 pages: through registers, widened exactly (once for all waves); the next
        // tile's loads leave as this one's are stored.  With the keys go the scales of
        // keys and values, which X(i) reads.
        constexpr int RCH = D / 16;
        float* const scales = reinterpret_cast<float*>(dsm + TABS); // [tile % 4][keys, values][kBN]
        auto fresh_tid = [&]() RDNA_INLINE { // no addresses kept in registers
            int td = tid & 255;
            asm volatile("" : "+v"(td));
            return td;
        };
        int32_t ent[C::NCH];
        i4 raw[C::NCH];
        float ksc[C::NCH], vsc[C::NCH];
        auto load_entries = [&](int t) RDNA_INLINE {
            const int td = fresh_tid();
#pragma unroll
            for (int c = 0; c < C::NCH; c++) {
                const int e = ((t0 + t) * kBN + (256 * c + td) / RCH) >> p.c.lps;
                ent[c] = p.c.table[walk.b * p.c.table_s + min(e, p.c.width - 1)];
            }
        };
        auto load_raw = [&](int t) RDNA_INLINE {
            const int td = fresh_tid();
            const char* const base = second ? kbase : vbase;
            const int64_t sp = second ? p.c.k_sp : p.c.v_sp;
            const int64_t st = second ? p.c.k_st : p.c.v_st;
#pragma unroll
            for (int c = 0; c < C::NCH; c++) {
                const int key = (t0 + t) * kBN + (256 * c + td) / RCH;
                const bool seen = key >= item.lo && key <= item.hi;
                const int64_t pg = (uint32_t)ent[c] < (uint32_t)p.c.pages ? ent[c] : 0;
                const int64_t off = (uint32_t)key & page_mask;
                raw[c] = *reinterpret_cast<const i4*>(base + pg * sp + off * st + 16 * (td % RCH));
                if (second) {
                    const float a = p.c.ks[pg * p.c.ks_sp + off * p.c.ks_st + h * p.c.ks_sh];
                    const float b = p.c.vs[pg * p.c.vs_sp + off * p.c.vs_st + h * p.c.vs_sh];
                    ksc[c] = seen ? a : 0.0f;
                    vsc[c] = seen ? b : 0.0f;
                }
            }
        };
        auto stage_int8 = [&](int t) RDNA_INLINE {
            const int td = fresh_tid();
#pragma unroll
            for (int c = 0; c < C::NCH; c++) {
                const int r = (256 * c + td) / RCH;
                const int cl = 2 * (td % RCH);
                // beyond the last tile the slots are free and hold rows of any page
                char* const s = dsm + (second ? 0 : V_SLOTS) + (t & 1) * C::TILE_BYTES + r * C::RB;
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    char* const at = s + (((cl + x) ^ paged_swz<D>(r)) << 4);
                    const i2v in{raw[c][2 * x], raw[c][2 * x + 1]};
                    if (second) {
                        *reinterpret_cast<V8*>(at) = widen_int8<T>(in);
                    } else {
                        *reinterpret_cast<P8*>(at) = widen_int8<P>(in);
                    }
                }
                if (second && cl == 0) {
                    scales[(t & 3) * 2 * kBN + r] = ksc[c];
                    scales[(t & 3) * 2 * kBN + kBN + r] = vsc[c];
                }
            }
            load_raw(t + 1);
            load_entries(t + 2);
        };
        // keys or values of tile t: of eight waves the wave's kind
        auto stage = [&](bool values, int t) RDNA_INLINE {
            if constexpr (I8) {
                stage_int8(t);
            } else {
                stage_copies(values, t);
            }
        };

        // ---- prologue: K(0); its Q and entries, on their way since the last item
        if constexpr (!I8 || C::Q_LDS) {
            __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
            asm volatile("" ::: "memory");
        }
        if (nt > 0) {
            if constexpr (I8) {
                load_entries(0);
                load_raw(0);
                load_entries(1);
            }
            if (!C::SPLIT || second) {
                stage(false, 0);
            }
        }
        V8 qreg[C::NS];
#pragma unroll
        for (int s = 0; s < C::NS; s++) {
            if constexpr (C::Q_LDS) {
                qreg[s] = *reinterpret_cast<const V8*>(dsm + QS + wave * C::Q_BYTES + l32 * C::RB +
                                                       (((2 * s + g) ^ paged_swz<D>(l32)) << 4));
            } else {
                qreg[s] = *reinterpret_cast<const V8*>(q_row(walk, tok, head) + 32 * s + 16 * g);
            }
        }
#pragma unroll
        for (int s = 0; s < C::NS; s++) {
            qreg[s] = col_valid ? (p.q_sign < 0.0f ? -qreg[s] : qreg[s]) : V8{};
        }

        f16x oacc[C::NDT];
#pragma unroll
        for (int dt = 0; dt < C::NDT; dt++) {
            oacc[dt] = f16x{};
        }
        float m_run = -INFINITY, l_run = 0.0f;
        float p_run = 0.0f; // JOIN, 16-bit pages: the sum of the weights as the products take them
        f16x sacc[2] = {f16x{}, f16x{}};
        P8 pb[4] = {P8{}, P8{}, P8{}, P8{}};
        ValueScale vscale;

        // M(i): one stream of MFMAs, operands read ahead.  (At raised wave priority it
        // takes up to 5 % more time: D = 160, B2 Hq16 Hkv8 S2048, 127 us against 121.)  There
        // are two of it only, M(0) and the others (M(nt) computes an S of no use, of
        // whatever K's slot holds): with one for every case O and S take twice the registers.
        auto mfmas = [&](auto do_pv, int i) RDNA_INLINE {
            constexpr int NPV = decltype(do_pv)::value ? 4 * C::NDT : 0; // (u, dt)
            constexpr int NSK = 2 * C::NS;                               // (s, kt)
            const uint32_t k_slot = (uint32_t)(i & 1) * C::TILE_BYTES;
            const uint32_t v_slot = (uint32_t)((i + 1) & 1) * C::TILE_BYTES;
            uint32_t ka[C::KA], va[2 * C::VA];
            if constexpr (C::KEEP) {
#pragma unroll
                for (int x = 0; x < 2 * C::VA; x++) {
                    va[x] = va0[x];
                }
#pragma unroll
                for (int s = 0; s < C::KA; s++) {
                    ka[s] = ka0[s];
                }
            } else {
                int ln = lane;
                asm volatile("" : "+v"(ln));
                addresses(ln, ka, va);
            }
#pragma unroll
            for (int x = 0; x < 2 * C::VA; x++) {
                va[x] += v_slot;
            }
#pragma unroll
            for (int s = 0; s < C::KA; s++) {
                ka[s] += k_slot;
            }
            operand_stream<NPV + NSK, C::DEPTH>(
                [&](int j) -> h8 {
                    if (j < NPV) {
                        const int u = j / C::NDT, dt = j % C::NDT;
                        const int x = 2 * (dt % C::VA), on = 16 * u * C::RB + dt / C::VA * 16 * C::SWZ;
                        const h4 lo = lds_read_tr16(va[x] + on);
                        const h4 hi = lds_read_tr16(va[x + 1] + on);
                        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    }
                    const int s = (j - NPV) >> 1, kt = (j - NPV) & 1;
                    return lds_read<h8>(ka[s % C::KA] + 32 * kt * C::RB + s / C::KA * 16 * C::SWZ);
                },
                [&](int j, h8 a) {
                    if (j < NPV) {
                        const int u = j / C::NDT, dt = j % C::NDT;
                        oacc[dt] = paged_mfma<P>(__builtin_bit_cast(P8, a), pb[u], oacc[dt]);
                    } else {
                        const int s = (j - NPV) >> 1, kt = (j - NPV) & 1;
                        sacc[kt] = paged_mfma<T>(__builtin_bit_cast(V8, a), qreg[s], s == 0 ? f16x{} : sacc[kt]);
                    }
                });
            // (the priority is zero already) keeps the softmax's instructions behind the last
            // product.  us with / without, causal S2048: B2 Hq32 Hkv8 D64 67.7 / 68.7, B2 Hq16 Hkv8
            // D256 144.7 / 142.7, D96 to D224 within 1 %
            __builtin_amdgcn_s_setprio(0);
        };
        auto softmax = [&](int i) RDNA_INLINE {
            const int kt0 = (t0 + i) * kBN;
            if constexpr (I8) {
                const f4* sc = reinterpret_cast<const f4*>(scales + (i & 3) * 2 * kBN) + g;
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const f4 ks = sc[2 * x];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        sacc[x >> 2][4 * (x & 3) + e] *= ks[e];
                    }
                }
            }
            if (tile_class(cls, t0 + i) != 1) { // a tile that the wave's rows do not see: all of it
                const int a = row_lo - kt0 - 4 * g;
                const int bnd = row_hi - kt0 - 4 * g;
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    const int off = 32 * (e >> 4) + 8 * ((e & 15) >> 2) + (e & 3);
                    sacc[e >> 4][e & 15] = (off < a || off > bnd) ? -INFINITY : sacc[e >> 4][e & 15];
                }
            }
            if (kt0 + kBN > tree_from) {
                tree_mask_scores<2>(sacc, tree_row, tree_n, prefix, kt0 + 4 * g);
            }
            const float mx = scores_max(sacc);
            const float m_new = fmaxf(m_run, mx * p.scale_log2e);
            const bool grow = m_new > m_run + kRescale;
            if (wave_any(grow)) {
                const float alpha = grow ? fast_exp2(m_run - m_new) : 1.0f;
                if (grow) {
                    m_run = m_new;
                }
                l_run *= alpha;
                if constexpr (JOIN && !I8) {
                    p_run *= alpha;
                }
#pragma unroll
                for (int dt = 0; dt < C::NDT; dt++) {
                    oacc[dt] *= alpha;
                }
            }
            const float m_use = (m_run == -INFINITY) ? 0.0f : m_run;
            float ps[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (I8) {
                float pv[32];
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    pv[e] = fast_exp2(fmaf(sacc[e >> 4][e & 15], p.scale_log2e, -m_use));
                    ps[e & 3] += pv[e];
                }
                const f4* sc = reinterpret_cast<const f4*>(scales + (i & 3) * 2 * kBN + kBN) + g;
                f4 vs[8];
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    vs[x] = sc[2 * x];
                }
                vscale.weigh<8>(pv, vs, oacc);
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    pb[e >> 3][e & 7] = (P)pv[e];
                }
            } else {
                float pr[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int x = 8 * u + e;
                        const float w = fast_exp2(fmaf(sacc[x >> 4][x & 15], p.scale_log2e, -m_use));
                        pb[u][e] = (P)w;
                        if constexpr (JOIN) { // the log-sum-exp is of the weights before they are rounded
                            ps[u] += w;
                        }
                    }
                    pr[u] = sum8<P>(pb[u], 0.0f); // of the weights as the products take them
                    if constexpr (!JOIN) {
                        ps[u] = pr[u];
                    }
                }
                if constexpr (JOIN) {
                    p_run += (pr[0] + pr[1]) + (pr[2] + pr[3]);
                }
            }
            l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        };

        // Every wave's copies (LDS stores) of the tiles to be read have landed behind a
        // barrier, and every wave has read what the copies behind it overwrite.
        using Yes = std::true_type;
        using No = std::false_type;
        if (nt > 0) {
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
        }
        auto ahead = walk;
        ahead.next();
        odd ^= 1;
        if (ahead.more()) {
            prefetch(ahead, odd);
        }
        odd ^= 1;
        if (nt > 0) {
            if (!C::SPLIT || second) {
                stage(false, 1);
            }
            if (!C::SPLIT || !second) {
                stage(true, 0);
            }
            if (active) {
                mfmas(No{}, 0);
            }
            for (int i = 0; i < nt; i++) {
                if (active) {
                    softmax(i);
                }
                if constexpr (!I8) {
                    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0)); // its copies of K(i + 1), V(i)
                }
                __syncthreads();
                if (!C::SPLIT || second) {
                    stage(false, i + 2);
                }
                if (!C::SPLIT || !second) {
                    stage(true, i + 1);
                }
                if (active) {
                    mfmas(Yes{}, i + 1);
                }
            }
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads(); // the next item's copies overwrite the slots
        }

        const float l_tot = pair_sum(l_run);
        float unit = I8 ? vscale.factor() : 1.0f; // of O
        if constexpr (JOIN && !I8) {
            // O over the sum of the weights that made it, so that their rounding cancels where few
            // keys count; l goes on to the log-sum-exp and weighs the parts
            const float p_tot = pair_sum(p_run);
            unit = p_tot > 0.0f ? l_tot / p_tot : 1.0f;
        }
        if (JOIN && whole) {
            const int64_t row = (int64_t)(seq.q0 + tok) * join.Hq + head;
            if (l_tot == 0.0f) { // as below
#pragma unroll
                for (int dt = 0; dt < C::NDT; dt++) {
                    oacc[dt] = f16x{};
                }
            }
            if (col_valid) {
                // addresses with the lane's part in them: as offsets of each access they would
                // be kept over the loop
                typedef __attribute__((address_space(1))) f4 g_f4;
                const PagedRowOut out = paged_row_out(join, row, m_run, l_tot);
                const float own = out.own * unit;
                const uint64_t at = 4 * (uint64_t)(row * D + 4 * g);
                const uint64_t pre = reinterpret_cast<uint64_t>(join.pre_o) + at;
                const uint64_t raw = reinterpret_cast<uint64_t>(join.raw_o) + at;
                char* const orow = p.o + (int64_t)(seq.q0 + tok) * p.o_st + head * p.o_sh + 8 * g;
                const bool with_pre = join.pre_o != nullptr && out.pre != 0.0f;
#pragma unroll
                for (int dt = 0; dt < C::NDT; dt++) {
#pragma unroll
                    for (int qq = 0; qq < 4; qq++) {
                        f4 x = f4{oacc[dt][4 * qq], oacc[dt][4 * qq + 1], oacc[dt][4 * qq + 2],
                                  oacc[dt][4 * qq + 3]} * own;
                        const int d = 32 * dt + 8 * qq;
                        if (with_pre) {
                            x += *reinterpret_cast<const g_f4*>(pre + 4 * d) * out.pre;
                        }
                        if (join.raw_o != nullptr) {
                            *reinterpret_cast<g_f4*>(raw + 4 * d) = x;
                        } else {
                            *reinterpret_cast<V4*>(orow + 2 * d) = __builtin_convertvector(x, V4);
                        }
                    }
                }
                if (g == 0) {
                    paged_store_lse(join, out, row);
                }
            }
        } else if (whole) {
            const float inv = l_tot > 0.0f ? unit / l_tot : 0.0f;
            if (l_tot == 0.0f) { // no key seen: weights of zero, of values that need not be finite
#pragma unroll
                for (int dt = 0; dt < C::NDT; dt++) {
                    oacc[dt] = f16x{};
                }
            }
            if (col_valid) {
                char* const orow = p.o + (int64_t)(seq.q0 + tok) * p.o_st + head * p.o_sh;
#pragma unroll
                for (int dt = 0; dt < C::NDT; dt++) {
#pragma unroll
                    for (int qq = 0; qq < 4; qq++) {
                        const f4 x = f4{oacc[dt][4 * qq], oacc[dt][4 * qq + 1], oacc[dt][4 * qq + 2],
                                        oacc[dt][4 * qq + 3]} * inv;
                        *reinterpret_cast<V4*>(orow + 2 * (32 * dt + 8 * qq + 4 * g)) = __builtin_convertvector(x, V4);
                    }
                }
            }
        } else {
            const int64_t slot = walk.slot();
            if (col_valid) {
                store_partial<C::NDT>(oacc, m_run, l_tot, g == 0, p.part_o, p.part_ml, slot * p.slot_rows + col, D, 0, g,
                                      [&](int) { return f4{unit, unit, unit, unit}; });
            }
            if (walk.begin() == 0) {
                rec = PagedRecord{n_rows, seq.q0, r0, h, walk.last_wg(), {}};
            }
        }
        walk.next();
        odd ^= 1;
    }
    if (tid == 0) {
        p.records[walk.part.wg] = rec;
    }
