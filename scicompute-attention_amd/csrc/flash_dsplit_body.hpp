// The body of the split-dims kernel (flash_dsplit.hip) and of its form over pages (paged_dsplit.hip), for
// inclusion in a kernel that has the template parameters E, D, kCausal and kDen, constants kCut and kPaged
// (packed rows of one sequence over the pages of its keys), and p, num_q_tiles, sp and job. (As a device
// function it compiles to other code: D 256, 16 heads x 4096 keys causal 128 -> 132 us.)
//
// Whatever is added here has to fit the registers: a copy or a reload that the compiler puts right before an
// inline-asm MFMA is read too early (the two wait states after a VALU write are not in the code), and a spill
// of an LDS read's result stores what was there before. Neither the plain nor the paged kernel has any.

    using G = DsplitGeom<D>;
    using M = Mfma<E>;
    using A = MfmaAsm<E>;
    using vec8 = typename E::vec8;
    constexpr int BN = G::BN;
    constexpr int BM = G::BM;
    constexpr int RB = G::ROW_BYTES;
    constexpr int kPagedRowsPerWave = BN / G::WAVES;  // 8
    // (see the wide kernel)
    constexpr float kBias = kPaged && std::is_same_v<E, F16> ? 7.0f : 0.0f;

    extern __shared__ __align__(16) uint8_t lds8[];
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int lane = tid % kWave;
    const int lr = lane & 31;
    const int hh = lane >> 5;
    const int rg = wave & 1;   // rows 64*rg .. +64 of the row tile
    const int dh = wave >> 1;  // QK: rows 32*dh of those; PV: dims D/2*dh .. +D/2

    const int pack = kCut ? sp.pack : 1;
    const int splits = kPaged ? job.splits : kCut ? sp.splits : 1;
    int tile_linear = 0, b_ = 0, unit = 0;
    int split = 0;
    if constexpr (kPaged) {
        unit = job.h_kv;
        split = job.split;
    } else {
        XcdOrder(p, static_cast<uint32_t>(p.num_heads) / static_cast<uint32_t>(pack), &tile_linear, &b_,
                 &unit);
    }
    if (!kPaged && splits > 1) {
        split = tile_linear % splits;
        tile_linear /= splits;
    }
    const int64_t b = b_;
    const int64_t h0 = static_cast<int64_t>(unit) * pack;  // first query head
    const int64_t h_kv =
        static_cast<int>(h0) / (static_cast<int>(p.num_heads) / static_cast<int>(p.num_kv_heads));
    const int qt = kPaged ? job.tile : kCausal ? (num_q_tiles - 1 - tile_linear) : tile_linear;
    const int seq_q = kPaged ? job.q_count : static_cast<int>(p.seq_q);
    const int64_t tok_q = kPaged ? job.q_first : 0;
    int seq_kv = kPaged ? job.keys : static_cast<int>(p.seq_kv);
    int diag = static_cast<int>(p.diagonal);
    const float scale2 = p.scale * kLog2e;
    const float inv_scale2 = 1.0f / scale2;
    const int q0 = qt * BM;
    // This lane's rows, of the owned subtile and of the partner's: query position and head offset
    // within the unit.
    int qi[2], hl[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        qi[r] = q0 + 64 * rg + 32 * (dh ^ r) + lr;
        hl[r] = 0;
        if (pack > 1) {
            const int row = qi[r];
            qi[r] = static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(pack));
            hl[r] = row - qi[r] * pack;
        }
    }

    int n_tiles = (seq_kv + BN - 1) / BN;
    int n_plain = seq_kv / BN;
    if (kCausal) {
        const int q_first = pack > 1 ? q0 / pack : q0;
        const int q_last = pack > 1 ? (q0 + BM - 1) / pack : q0 + BM - 1;
        const int last_key = q_last + diag;
        const int causal_tiles = last_key < 0 ? 0 : last_key / BN + 1;
        if (causal_tiles < n_tiles) n_tiles = causal_tiles;
        const int plain = (q_first + diag + 1) / BN;
        if (plain < n_plain) n_plain = plain;
    }
    if (n_plain > n_tiles) n_plain = n_tiles;
    int64_t key0 = 0;
    const int64_t rows_all = p.batch * p.num_heads * seq_q;
    // Index of the owned (then the partner's) row among the states and the LSE.
    auto flat_of = [&](int r) __attribute__((always_inline)) -> int64_t {
        if constexpr (kPaged) return job.state + static_cast<int64_t>(qi[r]) * pack + hl[r];
        return (b * p.num_heads + h0 + hl[r]) * seq_q + qi[r];
    };
    const int64_t flat_own = flat_of(0);
    if (splits > 1) {
        // Key tiles [first, first + count): the keys, the causal diagonal and K/V start there.
        int first, count;
        SplitRange(n_tiles, splits, split, &first, &count);
        if (!kPaged && count == 0) {  // fewer key tiles than splits: a state that the merge skips
            if (hh == 0 && qi[0] < seq_q) {
                float* ml = sp.part_ml + 2 * (split * rows_all + flat_own);
                ml[0] = neg_inf();
                ml[1] = 0.0f;
            }
            return;
        }
        key0 = static_cast<int64_t>(first) * BN;
        seq_kv = min(seq_kv - first * BN, count * BN);
        diag -= first * BN;
        n_tiles = count;
        n_plain = max(0, min(n_plain - first, count));
        // (paged: a range without keys runs through with every score masked, and leaves zeros)
        if (kPaged && count == 0) seq_kv = 0;
    }

    // ---- DMA (buffer resources bounded at the last row any row of this tile attends) ----
    const uint8_t* k_bytes = reinterpret_cast<const uint8_t*>(
        static_cast<const uint16_t*>(p.k) + b * p.k_sb + h_kv * p.k_sh + (kPaged ? 0 : key0) * p.k_ss);
    const uint8_t* v_bytes = reinterpret_cast<const uint8_t*>(
        static_cast<const uint16_t*>(p.v) + b * p.v_sb + h_kv * p.v_sh + (kPaged ? 0 : key0) * p.v_ss);
    const int k_row_bytes = static_cast<int>(p.k_ss) * 2;
    const int v_row_bytes = static_cast<int>(p.v_ss) * 2;
    const int rows = min(seq_kv, n_tiles * BN);
    const int k_records = (rows - 1) * k_row_bytes + RB;
    const int v_records = (rows - 1) * v_row_bytes + RB;
    uint32_t dma_koff[G::IPW], dma_voff[G::IPW];
#pragma unroll
    for (int i = 0; i < G::IPW; ++i) {
        const int P = (wave * G::IPW + i) * kWave + lane;
        const int row = P / G::CPR;
        const int pos = P % G::CPR;
        const int from = kPaged ? row - wave * kPagedRowsPerWave : row;  // paged: in the wave's rows
        dma_koff[i] = from * k_row_bytes + (pos ^ SwzK<D>(row)) * 16;
        dma_voff[i] = from * v_row_bytes + (pos ^ SwzV<D>(row)) * 16;
    }
    // Paged: a wave copies 8 rows of every tile, which one page holds; its id is asked for a step ahead.
    const int page_key0 = static_cast<int>(key0);
    const PagedKeys pages(job);
    if constexpr (kPaged) {
        // Tiles from the first page on that is not mapped are masked. (n_plain is negative where the first rows
        // come before the first key: more new tokens than keys.)
        n_plain = max(0, min(n_plain, (FirstHole(pages, job.table, page_key0, page_key0 + rows) - page_key0) / BN));
    }
    auto rows_of = [&](int t, int id) __attribute__((always_inline)) -> PagedRows {
        return RowsAt(pages, page_key0 + t * BN + wave * kPagedRowsPerWave, id, kPagedRowsPerWave, page_key0 + rows);
    };
    auto own_id = [&](int t) __attribute__((always_inline)) -> int {
        return pages.id(page_key0 + t * BN + wave * kPagedRowsPerWave);
    };
    // Holes of tile t (keys on pages that are not mapped): bit g for keys 8 g .. + 8.
    struct Ids {
        int of[4];
    };
    auto ids_of = [&](int t) __attribute__((always_inline)) -> Ids {
        Ids ids;
#pragma unroll
        for (int g = 0; g < 4; ++g) ids.of[g] = pages.id(page_key0 + t * BN + 8 * g);
        return ids;
    };
    auto holes_of = [&](int t, const Ids& ids) __attribute__((always_inline)) -> int {
        int holes = 0;
#pragma unroll
        for (int g = 0; g < 4; ++g) holes |= pages.hole(page_key0 + t * BN + 8 * g, ids.of[g]) ? 1 << g : 0;
        return holes;
    };
    PagedRows rows_v{0, 0}, rows_mid{0, 0}, rows_k{0, 0};  // of tiles t + 4, t + 5 and t + 6 in step t
    int id_own = 0;
    Ids tile_ids{};
    // DMA instruction i of this wave's share of K tile t (into K slot t & 3) or V tile t.
    auto dma_k = [&](int i, int slot, int t) __attribute__((always_inline)) {
        if constexpr (kPaged) {
            DmaRowsToLds<RB>(k_bytes, k_row_bytes, rows_k, lds8 + slot * G::TILE_BYTES + (wave * G::IPW + i) * 1024,
                             dma_koff[i]);
            return;
        }
        DmaToLds(k_bytes, k_records, lds8 + slot * G::TILE_BYTES + (wave * G::IPW + i) * 1024,
                 dma_koff[i], static_cast<uint32_t>(t * BN * k_row_bytes));
    };
    auto dma_v = [&](int i, int slot, int t) __attribute__((always_inline)) {
        if constexpr (kPaged) {
            DmaRowsToLds<RB>(v_bytes, v_row_bytes, rows_v,
                             lds8 + G::V_BASE + slot * G::TILE_BYTES + (wave * G::IPW + i) * 1024, dma_voff[i]);
            return;
        }
        DmaToLds(v_bytes, v_records,
                 lds8 + G::V_BASE + slot * G::TILE_BYTES + (wave * G::IPW + i) * 1024, dma_voff[i],
                 static_cast<uint32_t>(t * BN * v_row_bytes));
    };

    // ---- fragment addresses (LDS byte addresses of slot 0; slots are immediate offsets) ----
    const uint32_t lds_base = LdsAddr(lds8);
    constexpr int KP = KPeriod<D>();
    uint32_t k_addr[KP];
#pragma unroll
    for (int ks = 0; ks < KP; ++ks) {
        k_addr[ks] = lds_base + lr * RB + (((2 * ks) ^ hh ^ SwzK<D>(lr)) * 16);
    }
    const int grp = lane >> 4;
    const int sl = lane & 15;
    const int v_key = 4 * hh + (sl >> 2);
    const int v_chunk = 2 * (grp & 1) + ((sl & 3) >> 1);
    const int v_half = (sl & 1) * 8;
    uint32_t v_addr[G::DT];
#pragma unroll
    for (int dt = 0; dt < G::DT; ++dt) {
        v_addr[dt] = lds_base + G::V_BASE + v_key * RB +
                     (((4 * (dh * G::DT + dt) + v_chunk) ^ SwzV<D>(v_key)) * 16) + v_half;
    }
    // P fragments: [parity][wave][k-step][lane] of 16 bytes; own slot to write, partner's to read.
    const uint32_t p_own = lds_base + G::P_BASE + wave * 2048 + lane * 16;
    const uint32_t p_partner = lds_base + G::P_BASE + (wave ^ 2) * 2048 + lane * 16;
    // Rescale factors [parity][wave][32] and flags [parity][row group][dh] (the tile they are for).
    float* const s_alpha = reinterpret_cast<float*>(lds8 + G::ALPHA_BASE);
    int* const s_flag = reinterpret_cast<int*>(lds8 + G::FLAG_BASE);
    const uint32_t flag_addr = lds_base + G::FLAG_BASE + rg * 8;

    floatx16 o[2][G::DT];  // the owned subtile's rows, then the partner's
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int dt = 0; dt < G::DT; ++dt) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[r][dt][i] = 0.0f;
            PinAgpr(o[r][dt]);
        }
    }
    RowState rs;
    float l2 = 0.0f;  // second half of the denominator (two addition chains)
    float lw = 0.0f;  // the rounded weights' sum beside the unrounded one (kRoundedAndUnrounded)
    ResetRow(rs);

    vec8 kf[G::KS];           // K fragments of the next QK
    vec8 va[2][2 * G::DT];    // V^T fragments by tile parity
    auto read_k1 = [&]<int SLOT, int ks>() __attribute__((always_inline)) {
        ReadB128Asm<SLOT * G::TILE_BYTES + (ks / KP) * KP * 32>(kf[ks], k_addr[ks % KP]);
    };
    // Transposed V read i (of 4*DT) of the V tile in slot SLOT into buffer VB.
    auto read_v1 = [&]<int SLOT, int VB, int i>() __attribute__((always_inline)) {
        constexpr int dt = i / 4;
        constexpr int part = i % 4;
        const uint2 r = TrReadAsm<SLOT * G::TILE_BYTES + part * 8 * RB>(v_addr[dt]);
        uint4 w = __builtin_bit_cast(uint4, va[VB][2 * dt + part / 2]);
        if constexpr (part % 2 == 0) {
            w.x = r.x;
            w.y = r.y;
        } else {
            w.z = r.x;
            w.w = r.y;
        }
        va[VB][2 * dt + part / 2] = __builtin_bit_cast(vec8, w);
    };

    // Masking of the owned scores of key tile t (uniform `masked`), and the lane's maximum.
    auto mask_max = [&](floatx16& sr, int t, bool masked, int holes) __attribute__((always_inline)) -> float {
        if (masked) {
            const int kbase = t * BN + 4 * hh;
            const int lim = kCausal ? min(seq_kv - 1, qi[0] + diag) : seq_kv - 1;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = kbase + 8 * (i / 4) + (i % 4);
                sr[i] = key > lim || (kPaged && ((holes >> (i / 4)) & 1)) ? neg_inf() : sr[i];
            }
        }
        return Max16(sr);
    };
    // The owner's decision for tile t with raw lane maximum lm; publishes the factors of O.
    auto decide = [&](float lm, int t, int par) __attribute__((always_inline)) {
        if (__builtin_amdgcn_ballot_w64(lm > rs.thr) == 0) return;
        const float cmax = HalfMax(lm) * scale2;  // row maximum, log2 units
        const bool grow = cmax > rs.m + (kRescaleSlack + kBias);
        const float m_new = grow ? cmax - kBias : rs.m;
        const float alpha = grow ? fast_exp2(rs.m - m_new) : 1.0f;  // 0 when m was -inf
        rs.m = m_new;
        rs.l *= alpha;
        l2 *= alpha;
        lw *= alpha;
        rs.thr = (m_new + (kRescaleSlack + kBias)) * inv_scale2;
        rs.neg_mu = (m_new == neg_inf()) ? 0.0f : -m_new;
        if (hh == 0) s_alpha[(par * 4 + rg * 2 + dh) * 32 + lr] = alpha;
        if (lane == 0) s_flag[par * 4 + rg * 2 + dh] = t;
    };
    // O of both subtiles by the factors published for tile t (flags f of subtiles 0 and 1).
    auto apply = [&](uint2 f, int t, int par) __attribute__((always_inline)) {
        const int f0 = __builtin_amdgcn_readfirstlane(static_cast<int>(f.x));
        const int f1 = __builtin_amdgcn_readfirstlane(static_cast<int>(f.y));
        if (f0 != t && f1 != t) return;
        SettleO(o);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int sub = dh ^ r;
            const float published = s_alpha[(par * 4 + rg * 2 + sub) * 32 + lr];
            const float alpha = (sub == 0 ? f0 : f1) == t ? published : 1.0f;
#pragma unroll
            for (int dt = 0; dt < G::DT; ++dt) {
                Fence();  // one O tile at a time through VGPRs
#pragma unroll
                for (int i = 0; i < 16; ++i) o[r][dt][i] *= alpha;
                PinAgpr(o[r][dt]);
            }
            Fence();
        }
        asm volatile("s_nop 4");
    };
    // The VALU operations that turn the owned scores into P (SoftmaxOp); op(n, ...) runs the n-th.
    constexpr int kOps = SoftmaxOps(kDen);
    auto op = [&](int n, floatx16& s, uint32_t (&pw)[8]) __attribute__((always_inline)) {
        const int c = SoftmaxOp(kDen, n);
        if (c < 16) {
            s[c] = fmaf(s[c], scale2, rs.neg_mu);
        } else if (c < 32) {
            s[c - 16] = fast_exp2(s[c - 16]);
        } else if (c < 40) {
            pw[c - 32] = M::pack(s[2 * (c - 32)], s[2 * (c - 32) + 1]);
        } else if (c >= 56) {
            float& sum = kDen == kRoundedAndUnrounded ? lw : c % 2 == 0 ? rs.l : l2;
            sum = M::sum2(pw[c - 56], sum);
        } else if (c % 2 == 0) {
            rs.l += s[c - 40];
        } else {
            l2 += s[c - 40];
        }
    };
    auto pack_p = [&](const uint32_t (&pw)[8], vec8 (&pb)[2]) __attribute__((always_inline)) {
        pb[0] = __builtin_bit_cast(vec8, make_uint4(pw[0], pw[1], pw[2], pw[3]));
        pb[1] = __builtin_bit_cast(vec8, make_uint4(pw[4], pw[5], pw[6], pw[7]));
    };
    auto write_p = [&]<int PAR>(const vec8 (&pb)[2]) __attribute__((always_inline)) {
        WriteB128Asm<PAR * 8192>(p_own, pb[0]);
        WriteB128Asm<PAR * 8192 + 1024>(p_own, pb[1]);
    };

    // ---- prologue: S(0) -> P(0), S(1); K(2) and V(0) fragments. Issue order: K(0), K(1), then
    //      (K(t+2), V(t)) as in the steps ----
    PagedRows first_rows[6];  // paged: of tiles 0 to 5
    int holes0 = 0, holes1 = 0;
    if constexpr (kPaged) {
        int ids[6];
#pragma unroll
        for (int i = 0; i < 6; ++i) ids[i] = own_id(i);
        const Ids ids0 = ids_of(0), ids1 = ids_of(1);
        id_own = own_id(6);
#pragma unroll
        for (int i = 0; i < 6; ++i) first_rows[i] = rows_of(i, ids[i]);
        holes0 = holes_of(0, ids0);
        holes1 = holes_of(1, ids1);
    }
    auto issue = [&](int t_k, int t_v) __attribute__((always_inline)) {
        if constexpr (kPaged) {
            rows_k = first_rows[t_k];
            rows_v = first_rows[t_v];
        }
#pragma unroll
        for (int i = 0; i < G::IPW; ++i) dma_k(i, t_k & 3, t_k);
#pragma unroll
        for (int i = 0; i < G::IPW; ++i) dma_v(i, t_v & 3, t_v);
    };
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        if constexpr (kPaged) rows_k = first_rows[t];
#pragma unroll
        for (int i = 0; i < G::IPW; ++i) dma_k(i, t, t);
    }
    // Q fragments of the owned subtile (B operand of S^T = K Q^T). Rows past seq_q repeat the last
    // one (their results are not stored); pinned only after the other tiles' DMAs are issued, so that
    // nothing waits for them but the first QK.
    vec8 qf[G::KS];
    {
        const uint16_t* q_row = static_cast<const uint16_t*>(p.q) + b * p.q_sb +
                                (h0 + hl[0]) * p.q_sh +
                                (tok_q + min(qi[0], seq_q - 1)) * p.q_ss + 8 * hh;
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks) {
            qf[ks] = __builtin_bit_cast(vec8, *reinterpret_cast<const uint4*>(q_row + 16 * ks));
        }
    }
    issue(2, 0);
    issue(3, 1);
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) PinAgpr(qf[ks]);
    if (tid < 8) s_flag[tid] = 0;  // tile 0 is never rescaled for
    WaitVm<4 * G::IPW>();          // K(0), K(1)
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_s_barrier();
    floatx16 s0, s1;
    vec8 pb0[2], pb1[2];
    auto qk_all = [&](floatx16& s) __attribute__((always_inline)) {
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks) WaitLgkmTied<0>(kf[ks]);
        A::first_v(s, kf[0], qf[0]);
#pragma unroll
        for (int ks = 1; ks < G::KS; ++ks) A::acc_v(s, kf[ks], qf[ks]);
        asm volatile("s_nop 15\n\ts_nop 15" : "+v"(s));  // complete, and kf has been read
    };
    StaticFor<G::KS>([&](auto ks) __attribute__((always_inline)) { read_k1.template operator()<0, ks>(); });
    qk_all(s0);
    StaticFor<G::KS>([&](auto ks) __attribute__((always_inline)) { read_k1.template operator()<1, ks>(); });
    {
        const float lm = mask_max(s0, 0, n_plain == 0, holes0);
        decide(lm, 0, 0);  // O is zero: the factors published for tile 0 are never read
    }
    qk_all(s1);
    {
        uint32_t pw[8];
#pragma unroll
        for (int n = 0; n < kOps; ++n) op(n, s0, pw);
        pack_p(pw, pb0);
        write_p.template operator()<0>(pb0);
        const float lm = mask_max(s1, 1, n_plain <= 1, holes1);
        decide(lm, 1, 1);
    }
    WaitVm<2 * G::IPW>();  // K(2), V(0)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    issue(4, 2);  // K slots 0 and 1 were read before the barrier
    issue(5, 3);
    StaticFor<G::KS>([&](auto ks) __attribute__((always_inline)) { read_k1.template operator()<2, ks>(); });
    StaticFor<4 * G::DT>([&](auto i) __attribute__((always_inline)) { read_v1.template operator()<0, 0, i>(); });
    WaitVm<4 * G::IPW>();  // K(3), V(1)
    WaitLgkmTied<0>(kf[G::KS - 1]);
    __builtin_amdgcn_s_barrier();

    // One step for key tile t (S = t & 3). On entry kf holds K(t+2)'s fragments, va[t & 1] V(t)'s,
    // s_in the masked scores of tile t+1 (its decision made), pb_in the owned P(t); the partner's
    // P(t) and the flags of tile t+1 are in LDS; K(t+3) and V(t+1) have landed.
    //   A  QK(t+2) | partner's P(t), flags(t+1), V(t+1)'s fragments; exponentials of tile t+1
    //   B  PV(t), own subtile first | write P(t+1), mask and maximum of tile t+2, K(t+3)'s fragments
    //   then the factors of tile t+1 to O, the decision for tile t+2, the waits and the barrier.
    auto step = [&]<bool kMaskable, int S>(int t, floatx16& s_in, floatx16& s_out, vec8 (&pb_in)[2],
                                           vec8 (&pb_out)[2]) __attribute__((always_inline)) {
        constexpr int VB = S & 1;
        constexpr int NPV = 4 * G::DT;  // PV MFMAs: 2 subtiles x DT x 2 k-steps
        vec8 pbx[2];
        uint2 flags;
        uint32_t pw[8];
        int next_holes = 0;
        if constexpr (kPaged) {
            // The page ids asked for a step ago, and the next ones: the scalar loads are back before the
            // step's last wait, so that their use costs none.
            rows_k = rows_of(t + 6, id_own);
            id_own = own_id(t + 7);
            if constexpr (kMaskable) {
                next_holes = holes_of(t + 2, tile_ids);
                tile_ids = ids_of(t + 3);
            }
        }
        // ---- A ----
        constexpr int kOpsA = (kOps + G::KS - 1) / G::KS;
        constexpr int kVReads = (4 * G::DT + G::KS - 4) / (G::KS - 3);
        StaticFor<G::KS>([&](auto ks) __attribute__((always_inline)) {
            if constexpr (ks == 0) {
                A::first_v(s_out, kf[0], qf[0]);
            } else {
                A::acc_v(s_out, kf[ks], qf[ks]);
            }
            Fence();
            if constexpr (ks == 0) {
                ReadB128Asm<VB * 8192>(pbx[0], p_partner);
                ReadB128Asm<VB * 8192 + 1024>(pbx[1], p_partner);
                ReadB64Asm<(VB ^ 1) * 16>(flags, flag_addr);
            }
            StaticFor<kVReads>([&](auto q) __attribute__((always_inline)) {
                constexpr int i = (ks - 1) * kVReads + q;
                if constexpr (ks >= 1 && i < 4 * G::DT) {
                    read_v1.template operator()<(S + 1) & 3, VB ^ 1, i>();
                }
            });
#pragma unroll
            for (int q = 0; q < kOpsA; ++q) {
                if (ks * kOpsA + q < kOps) op(ks * kOpsA + q, s_in, pw);
            }
            if constexpr (ks % 4 == 2 && ks / 4 < G::IPW) dma_k(ks / 4, (S + 2) & 3, t + 6);
            Fence();
        });
        pack_p(pw, pb_out);
        // The partner's P and the flags have arrived (every read of region A, in order).
        WaitLgkmTied<0>(pbx[0]);
        WaitLgkmTied<0>(pbx[1]);
        WaitLgkmTied<0>(flags);
        // ---- B ----
        float lm = neg_inf();
        StaticFor<NPV>([&](auto i) __attribute__((always_inline)) {
            constexpr bool kOwn = i < NPV / 2;
            constexpr int f = i % (NPV / 2);  // fragment 2*dt + k-step
            if constexpr (kOwn) {
                A::acc_a(o[0][f / 2], va[VB][f], pb_in[f % 2]);
            } else {
                A::acc_a(o[1][f / 2], va[VB][f], pbx[f % 2]);
            }
            Fence();
            if constexpr (i == 0) write_p.template operator()<VB ^ 1>(pb_out);
            if constexpr (i == 2) {
                asm volatile("s_nop 4");
                lm = mask_max(s_out, t + 2, kMaskable && t + 2 >= n_plain, next_holes);
            }
            if constexpr (i >= 2) {
                // KS K reads over the MFMAs 2 .. (kf was last read three MFMAs ago).
                constexpr int kPer = (G::KS + NPV - 4) / (NPV - 3);
                StaticFor<kPer>([&](auto q) __attribute__((always_inline)) {
                    constexpr int ks = (i - 2) * kPer + q;
                    if constexpr (ks < G::KS) read_k1.template operator()<(S + 3) & 3, ks>();
                });
            }
            if constexpr (i % 4 == 1 && i / 4 < G::IPW) dma_v(i / 4, S, t + 4);
            Fence();
        });
        if constexpr (kPaged) {
            rows_v = rows_mid;
            rows_mid = rows_k;
        }
        apply(flags, t + 1, VB ^ 1);
        decide(lm, t + 2, VB);
        Fence();
        // K(t+4) and V(t+2) landed (the groups of this step and the one before stay in flight);
        // fragment reads and LDS writes retired.
        WaitVm<4 * G::IPW>();
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(kf[G::KS - 1])::"memory");
        __builtin_amdgcn_s_barrier();
    };

    int t = 0;
    if constexpr (kPaged) {
        rows_v = first_rows[4];
        rows_mid = first_rows[5];
    }
    for (; t + 6 <= n_plain; t += 4) {
        step.template operator()<false, 0>(t, s1, s0, pb0, pb1);
        step.template operator()<false, 1>(t + 1, s0, s1, pb1, pb0);
        step.template operator()<false, 2>(t + 2, s1, s0, pb0, pb1);
        step.template operator()<false, 3>(t + 3, s0, s1, pb1, pb0);
    }
    if constexpr (kPaged) tile_ids = ids_of(t + 2);
    for (; t < n_tiles; t += 4) {
        step.template operator()<true, 0>(t, s1, s0, pb0, pb1);
        if (t + 1 >= n_tiles) break;
        step.template operator()<true, 1>(t + 1, s0, s1, pb1, pb0);
        if (t + 2 >= n_tiles) break;
        step.template operator()<true, 2>(t + 2, s1, s0, pb0, pb1);
        if (t + 3 >= n_tiles) break;
        step.template operator()<true, 3>(t + 3, s0, s1, pb1, pb0);
    }

    // ---- epilogue: share 1/l, normalise, store ----
    WaitVm<0>();
    SettleO(o);
    constexpr bool kBoth = kDen == kRoundedAndUnrounded;
    const float l_lse = HalfSum(rs.l + l2);
    const float l_tot = kBoth ? HalfSum(lw) : l_lse;
    if (splits > 1) {
        // The unnormalised state: both subtiles' O at the scale of their owner's m (and, with two
        // denominators, to the scale of the unrounded one, which the merge takes).
        if (hh == 0) {
            if (kBoth) s_alpha[(rg * 2 + dh) * 32 + lr] = l_tot > 0.0f ? l_lse / l_tot : 0.0f;
            if (qi[0] < seq_q) {
                *reinterpret_cast<float2*>(sp.part_ml + 2 * ((kPaged ? 0 : split * rows_all) + flat_own)) =
                    make_float2(rs.m, l_lse);
            }
        }
        if (kBoth) __syncthreads();
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float* dst = sp.part_o + ((kPaged ? 0 : split * rows_all) + flat_of(r)) * D + dh * (D / 2);
            const float to_l = kBoth ? s_alpha[(rg * 2 + (dh ^ r)) * 32 + lr] : 1.0f;
#pragma unroll
            for (int dt = 0; dt < G::DT; ++dt) {
                float a[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) a[i] = o[r][dt][i] * to_l;
                StorePartialTile(dst + 32 * dt, hh, qi[r] < seq_q, a);
            }
        }
        return;
    }
    if (hh == 0) {
        s_alpha[(rg * 2 + dh) * 32 + lr] = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
        if constexpr (kPaged) {
            if (qi[0] < seq_q && p.lse != nullptr) {
                // (the bits: compiled without regard to NaN, a comparison could take a NaN sum for none)
                const bool none = __builtin_bit_cast(uint32_t, l_lse) == 0;
                p.lse[(tok_q + qi[0]) * p.num_heads + h0 + hl[0]] =
                    none ? neg_inf() : (rs.m + __log2f(l_lse)) * kLn2;
            }
        } else if (qi[0] < seq_q && p.lse != nullptr) {
            p.lse[flat_own] = l_lse > 0.0f ? (rs.m + __log2f(l_lse)) * kLn2 : neg_inf();
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const float inv = s_alpha[(rg * 2 + (dh ^ r)) * 32 + lr];
        uint16_t* out_row = static_cast<uint16_t*>(p.out) + b * p.o_sb + (h0 + hl[r]) * p.o_sh +
                            (tok_q + qi[r]) * p.o_ss + dh * (D / 2);
#pragma unroll
        for (int dt = 0; dt < G::DT; ++dt) {
            float a[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) a[i] = o[r][dt][i] * inv;
            StoreTile<M>(out_row + 32 * dt, hh, qi[r] < seq_q, a);
        }
    }
