// The body of k_attend and attend_block (attend.h): `a` and `number` are their arguments, T, FMT, HD, RT, P16 and MODE
// their template's.
    constexpr bool EIGHT = FMT == RL_I8 || FMT == RL_F8, F32Q = sizeof(T) == 4;
    // Element types of the two products. 8-bit codes are exact in either; queries fit f16 scaled by a power of two
    // (below), weights times a value's step need bf16's range.
    using MK = std::conditional_t<FMT == RL_BF16, bhalf_t, half_t>;
    using MV = std::conditional_t<FMT == RL_F16, half_t, bhalf_t>;
    // f32 queries are split into parts that add up to them (24 bits in three bf16 parts, 22 in two of f16), and so are
    // the weights of f32 outputs. Those of 16-bit outputs are two parts too (16 or 22 bits): one alone, of 8 bits, cost as
    // much as the output's own rounding (0.0025 off f64 against 0.0017 over 64 int8 sequences), and a second product
    // hides behind the loads.
    constexpr int QP = !F32Q ? 1 : std::is_same_v<MK, bhalf_t> ? 3 : 2, PP = F32Q && std::is_same_v<MV, bhalf_t> ? 3 : 2;
    constexpr int ROWS = 16 * RT, VD = HD / 16, SIZE = EIGHT ? 1 : 2;
    constexpr int KC = HD * SIZE / 64;        // 64-byte chunks of a key
    constexpr int VW = VD * SIZE / 4;         // dwords of a value that a lane holds
    constexpr int STEPS = HD / 32;            // products a score tile
    constexpr float LIFT = FMT == RL_F16 ? ATTEND_LIFT : 0.0f; // weights up to 2^8: their second f16 parts stay normal
    constexpr bool Q_REGS = RT * QP * STEPS <= 4;
    constexpr int QS = HD + 8;
    constexpr size_t Q_BYTES = (size_t)QP * ROWS * QS * 2, O_BYTES = (size_t)ATTEND_WAVES * 16 * (HD + 4) * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES];
    __shared__ float mults[ROWS], maxima[ATTEND_WAVES][ROWS], sums[ATTEND_WAVES][ROWS];
    __shared__ bool last;

    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const uint32_t G = a.group;
    // Not written while the kernel runs: read through the scalar cache where the index is the wave's.
    typedef const __attribute__((address_space(4))) int32_t constant_i32;
    const constant_i32 *starts = (constant_i32 *)(uintptr_t)a.starts, *lens = (constant_i32 *)(uintptr_t)a.lens;
    // The first row of sequence or group i.
    const auto first_of = [&](uint32_t i) {
        if constexpr (MODE == ATTEND_PREFIX) {
            const int32_t at = min(max(((constant_i32 *)(uintptr_t)a.group_starts)[i], 0), (int32_t)a.group_end);
            return starts ? starts[at] : at;
        } else
            return starts ? starts[i] : (int32_t)i;
    };
    uint32_t s, head, part, block;
    if (a.packed) {
        const uint32_t y = number / 8, at = (y / ATTEND_RUN * 8 + number % 8) * ATTEND_RUN + y % ATTEND_RUN;
        const uint2 column = split_by(at, a.blocks, a.blocks_inv), of = split_by(column.x, a.cache.heads, a.heads_inv);
        const uint32_t b = column.y;
        part = of.x, head = of.y;
        if (part >= a.parts) return;
        // The last sequence whose row blocks begin at or before this one; no two begin at the same.
        const auto first_block = [&](uint32_t i) { return (uint32_t)min(max(first_of(i), 0), (int32_t)a.rows) * G / ROWS + i; };
        s = 0;
        for (uint32_t hi = a.seqs; hi - s > 1;) {
            const uint32_t mid = s + (hi - s) / 2;
            if (first_block(mid) <= b) s = mid;
            else hi = mid;
        }
        if (first_block(s) > b) return;
        block = b - first_block(s);
    } else {
        // The row blocks of one sequence, head and part are eight workgroups apart: on one XCD.
        const uint2 eight = split_by(number / 8, a.blocks, a.blocks_inv);
        const uint2 job = split_by(eight.x * 8 + number % 8, a.seqs * a.cache.heads, a.columns_inv);
        const uint2 of = split_by(job.y, a.cache.heads, a.heads_inv);
        block = eight.y, part = job.x, s = of.x, head = of.y;
        if (part >= a.parts) return;
    }
    const int32_t first = first_of(s);
    uint32_t shared_parts = 0; // of the sequence's prefix
    if constexpr (MODE == ATTEND_JOINED) {
        const constant_i32 *group_starts = (constant_i32 *)(uintptr_t)a.group_starts;
        if ((int32_t)s >= group_starts[0] && (int32_t)s < group_starts[a.group_end]) shared_parts = a.shared_parts;
    }
    const int64_t rows = MODE == ATTEND_PREFIX ? (int64_t)first_of(s + 1) - first : starts ? (int64_t)starts[s + 1] - first : 1;
    if (rows <= 0 || first < 0 || first + rows > a.rows) return; // no rows, or `starts` is not what it should be
    AttendSpan<MODE> span{max(lens[s], 0), (int32_t)rows, (int32_t)a.window}; // a negative length is none
    const uint32_t expanded = (uint32_t)span.n * G;
    const int32_t longest = span.end(span.n - 1);
    const uint32_t page = a.cache.page;
    // What the call's bounds or the page table do not cover is NaN, written once.
    if ((uint32_t)span.n > a.most_rows || span.len > (int64_t)a.max_len ||
        (longest > 0 && split_by(longest - 1, page, a.cache.page_inv).x >= a.table_width)) {
        if (part || block) return;
        const uint32_t dim = a.cache.dim;
        for (uint64_t i = tid; i < (uint64_t)expanded * dim; i += ATTEND_THREADS) {
            const uint32_t e = (uint32_t)(i / dim), d = (uint32_t)(i - (uint64_t)e * dim);
            const uint64_t row = first + e / G, qh = head * G + e % G;
            if constexpr (MODE == ATTEND_PREFIX) { // one part that is NaN, and no others
                if (d < a.shared_parts)
                    a.part_sum[(row * a.q_heads + qh) * a.stride + a.shared + d] = d ? make_float2(-INFINITY, 0.0f) : make_float2(0.0f, NAN);
                continue;
            }
            ((T *)a.out)[row * a.out_row + qh * a.out_head + d] = (T)NAN;
            if (d == 0 && a.lse) a.lse[row * a.q_heads + qh] = NAN;
        }
        return;
    }
    if (block >= (expanded + ROWS - 1) / ROWS) return;
    const uint32_t r0 = block * ROWS;
    const uint32_t count = min(expanded - r0, (uint32_t)ROWS);
    const auto by_group = [&](uint32_t e) { return split_by(e, G, a.group_inv); }; // (query row, query head of the group)
    const int32_t i0 = by_group(r0).x, i1 = by_group(r0 + count - 1).x; // query rows of the block
    const int32_t begin_min = span.begin(i0), begin_max = span.begin(i1), end_min = span.end(i0), end_max = span.end(i1);
    const bool mixed = begin_min != begin_max || end_min != end_max;
    const int32_t tile0 = begin_min / (int)ATTEND_TILE, tiles = (int32_t)((end_max + ATTEND_TILE - 1) / ATTEND_TILE) - tile0;
    const uint32_t parts = tiles > 0 ? split_by(tiles + a.part_tiles - 1, a.part_tiles, a.tiles_inv).x : 1; // of this block
    if (part >= parts) {
        if constexpr (MODE == ATTEND_PREFIX) // nothing here
            for (uint32_t i = tid; i < count; i += ATTEND_THREADS) {
                const uint2 e = by_group(r0 + i);
                a.part_sum[((uint64_t)(first + e.x) * a.q_heads + head * G + e.y) * a.stride + a.shared + part] = make_float2(-INFINITY, 0.0f);
            }
        return;
    }

    // The block's queries, a few values a thread; they go to LDS while the first tile is on its way.
    constexpr uint32_t TPR = ATTEND_THREADS / ROWS, EPT = HD / TPR;
    const uint32_t q_row = tid / TPR, q_at = tid % TPR * EPT;
    float x[EPT] = {};
    if (q_row < count) {
        const uint2 e = by_group(r0 + q_row);
        const T *q = (const T *)a.q + (uint64_t)(first + e.x) * a.q_row + (uint64_t)(head * G + e.y) * a.q_head;
#pragma unroll
        for (uint32_t j = 0; j < EPT; j += 4)
            if (q_at + j < a.cache.dim) { // dim is a multiple of 16
                float y[4];
                load_f32(q + q_at + j, a.wide, y);
#pragma unroll
                for (int c = 0; c < 4; c++) x[j + c] = y[c];
            }
    }

    const uint32_t col = lane % 16, quad = lane / 16;
    f32x4 O[RT][VD];
    float top[RT], total[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        top[rt] = -INFINITY, total[rt] = 0.0f;
#pragma unroll
        for (int m = 0; m < VD; m++) O[rt][m] = f32x4{0, 0, 0, 0};
    }

    const uint32_t dim_bytes = a.cache.dim * SIZE;
    const uint8_t *keys = (const uint8_t *)a.cache.keys, *values = (const uint8_t *)a.cache.values;
    const auto *table = (constant_i32 *)(uintptr_t)(a.pages + (uint64_t)s * a.table_width);
    const uint32_t pool = (uint32_t)(a.cache.slots / page);
    bool poison = false; // a page number that is none

    u32x4 kr[2][KC];
    uint32_t vr[8][VW];
    f32x4 ks[2], vs[2];

    // Where a tile's tokens lie. P16 (pages of a multiple of 16 tokens): each half of a tile lies in one page, at[u] is
    // its first vector. Else lane l has the vector of token l % 32. Tokens that no row sees, whose pages are not looked
    // up, are the nearest that some row does: what is loaded for them is masked, and no load is conditional.
    // Page numbers are fetched two tiles ahead, before the keys of the next: waiting for them waits for nothing newer.
    struct Place {
        uint64_t at[2];
    };
    struct Pages {
        uint32_t id[2];
    };
    auto in_sight = [&](int32_t t) {
        return (uint32_t)(P16 ? min(max(t, begin_min & ~15), (end_max - 1) & ~15) : min(max(t, begin_min), end_max - 1));
    };
    auto fetch = [&](int32_t t0) {
        Pages p{{0, 0}};
#pragma unroll
        for (int u = 0; u < (P16 ? 2 : 1); u++)
            p.id[u] = (uint32_t)table[split_by(in_sight(t0 + (P16 ? 16 * u : (int)(lane % 32))), page, a.cache.page_inv).x];
        return p;
    };
    auto place = [&](int32_t t0, const Pages &p) {
        Place w{{0, 0}};
#pragma unroll
        for (int u = 0; u < (P16 ? 2 : 1); u++) {
            const uint32_t t = in_sight(t0 + (P16 ? 16 * u : (int)(lane % 32)));
            poison |= p.id[u] >= pool;
            w.at[u] = ((uint64_t)(p.id[u] < pool ? p.id[u] : 0) * a.cache.heads + head) * page + split_by(t, page, a.cache.page_inv).y;
        }
        return w;
    };
    auto vector_at = [&](const Place &w, uint32_t token) -> uint64_t { // token of the tile
        if constexpr (P16) return w.at[token / 16] + token % 16;
        else return __shfl(w.at[0], token);
    };
    // Lanes past the head's end load its start: as keys they are zeroed before use, as values they are columns that are
    // not written.
    auto load_keys = [&](const Place &w) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint8_t *p = keys + (P16 ? w.at[u] * dim_bytes + col * dim_bytes : vector_at(w, 16 * u + col) * dim_bytes);
#pragma unroll
            for (uint32_t c = 0; c < KC; c++) {
                const uint32_t at = c * 64 + quad * 16;
                kr[u][c] = *(const u32x4 *)(p + (at < dim_bytes ? at : 0));
            }
            if constexpr (EIGHT) {
                if constexpr (P16) ks[u] = *(const f32x4 *)(a.cache.key_steps + w.at[u] + quad * 4);
                else
#pragma unroll
                    for (int i = 0; i < 4; i++) ks[u][i] = a.cache.key_steps[vector_at(w, 16 * u + quad * 4 + i)];
            }
        }
    };
    auto load_values = [&](const Place &w) {
        constexpr int PER = VW < 4 ? VW : 4;
        const uint32_t at = col * VW * 4 < dim_bytes ? col * VW * 4 : 0; // dim is a multiple of 16: a lane has all or none
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint64_t v = P16 ? w.at[j / 4] : vector_at(w, j / 4 * 16 + quad * 4 + j % 4);
            const uint8_t *p = values + (P16 ? v * dim_bytes + (quad * 4 + j % 4) * dim_bytes : v * dim_bytes) + at;
#pragma unroll
            for (int c = 0; c < VW; c += PER) {
                const vec<uint32_t, PER> x = *(const vec<uint32_t, PER> *)(p + c * 4);
#pragma unroll
                for (int e = 0; e < PER; e++) vr[j][c + e] = x[e];
            }
            if constexpr (EIGHT && !P16) vs[j / 4][j % 4] = a.cache.value_steps[v];
        }
        if constexpr (EIGHT && P16) {
#pragma unroll
            for (int u = 0; u < 2; u++) vs[u] = *(const f32x4 *)(a.cache.value_steps + w.at[u] + quad * 4);
        }
    };

    // The product with the values: for each of a lane's VD columns the eight tokens' values, column by column.
    auto multiply = [&](const u32x4 &v, const vec<MV, 8> (&w)[RT][PP], int column) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int p = 0; p < PP; p++)
                O[rt][column] = mfma(__builtin_bit_cast(vec<MV, 8>, v), w[rt][p], O[rt][column]);
    };
    // f(values of eight tokens, column) for each of a lane's columns.
    auto each_column = [&](auto f) {
        if constexpr (!EIGHT) {
#pragma unroll
            for (int c = 0; c < VW; c++) {
                u32x4 lo, hi;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    lo[j] = __builtin_amdgcn_perm(vr[2 * j + 1][c], vr[2 * j][c], 0x05040100u);
                    hi[j] = __builtin_amdgcn_perm(vr[2 * j + 1][c], vr[2 * j][c], 0x07060302u);
                }
                f(lo, 2 * c);
                f(hi, 2 * c + 1);
            }
        } else {
#pragma unroll
            for (int c = 0; c < VW; c++) {
                u32x4 x[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t lo = __builtin_amdgcn_perm(vr[2 * j + 1][c], vr[2 * j][c], 0x05010400u);
                    const uint32_t hi = __builtin_amdgcn_perm(vr[2 * j + 1][c], vr[2 * j][c], 0x07030602u);
                    x[0][j] = pair_bf16<FMT, false>(lo);
                    x[1][j] = pair_bf16<FMT, true>(lo);
                    x[2][j] = pair_bf16<FMT, false>(hi);
                    x[3][j] = pair_bf16<FMT, true>(hi);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) f(x[e], 4 * c + e);
            }
        }
    };

    const int32_t part_begin = tile0 + (int32_t)(part * a.part_tiles);
    const int32_t part_end = min(part_begin + (int32_t)a.part_tiles, tile0 + tiles);
    int32_t tile = part_begin + (int32_t)wave;
    Pages ahead{{0, 0}}; // of this wave's next tile
    if (tile < part_end) {
        // In the order of the loop's own loads: a wait in the loop has to hold for the first tile too.
        const int32_t t0 = tile * (int)ATTEND_TILE;
        const Pages now = fetch(t0);
        ahead = fetch((int32_t)(t0 + ATTEND_WAVES * ATTEND_TILE)); // may be past the last token, and past 2^31: any in sight
        const Place at = place(t0, now);
        __builtin_amdgcn_sched_barrier(0);
        load_keys(at);
        __builtin_amdgcn_sched_barrier(0);
        load_values(at);
        __builtin_amdgcn_sched_barrier(0);
    }
    // Queries into LDS in the type of the product. In f16 a row is scaled by the power of two that brings its largest
    // value to [1, 2), which costs nothing of its values down to 2^-24 of the largest.
    {
        MK *qs = (MK *)lds;
        float unit = 1.0f;
        if constexpr (std::is_same_v<MK, half_t>) {
            float m = 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < EPT; j++) m = fmaxf(m, fabsf(x[j]));
            m = group_max<TPR>(m);
            // 2^-e for m in [2^e, 2^(e+1)); the bounds keep it and its inverse normal.
            const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 100);
            const float down = __uint_as_float((uint32_t)(127 - e) << 23);
            unit = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (uint32_t j = 0; j < EPT; j++) x[j] *= down;
        }
#pragma unroll
        for (int p = 0; p < QP; p++)
#pragma unroll
            for (uint32_t j = 0; j < EPT; j++) {
                const MK y = (MK)x[j];
                qs[(p * ROWS + q_row) * QS + q_at + j] = y;
                x[j] -= (float)y;
            }
        if (tid % TPR == 0) mults[q_row] = a.scale * 1.44269504088896341f * unit;
    }
    __syncthreads();
    const MK *qs = (const MK *)lds;
    // Contraction order of a product: 16-bit keys 32 dims in order, 8-bit ones the first or second half of each lane's
    // 16 bytes. Queries follow it.
    auto q_fragment = [&](int rt, int p, int st) {
        const uint32_t d = EIGHT ? st / 2 * 64 + quad * 16 + st % 2 * 8 : st * 32 + quad * 8;
        return *(const vec<MK, 8> *)(qs + (p * ROWS + rt * 16 + col) * QS + d);
    };
    vec<MK, 8> qf[Q_REGS ? RT : 1][Q_REGS ? QP : 1][Q_REGS ? STEPS : 1];
    if constexpr (Q_REGS) {
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int p = 0; p < QP; p++)
#pragma unroll
                for (int st = 0; st < STEPS; st++) qf[rt][p][st] = q_fragment(rt, p, st);
    }
    float mult[RT];
    int32_t row_begin[RT], row_end[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const uint32_t r = rt * 16 + col;
        mult[rt] = mults[r];
        const int32_t i = r < count ? by_group(r0 + r).x : 0;
        row_begin[rt] = r < count ? span.begin(i) : begin_min; // rows past the block's see what any of it sees
        row_end[rt] = r < count ? span.end(i) : end_max;
    }
    // A tile; with `more` the next one's loads go out as their registers become free. That is known to the compiler, so
    // that a wait for this tile's values leaves the next one's keys on their way.
    auto step = [&](auto more) {
        constexpr bool MORE = decltype(more)::value;
        const int32_t t0 = tile * (int)ATTEND_TILE;
        f32x4 S[RT][2];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int rt = 0; rt < RT; rt++) S[rt][u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            vec<MK, 8> k[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if constexpr (EIGHT) {
                    const uint32_t x = kr[u][st / 2][st % 2 * 2], y = kr[u][st / 2][st % 2 * 2 + 1];
                    const u32x4 w = {pair_f16<FMT, false>(x), pair_f16<FMT, true>(x), pair_f16<FMT, false>(y), pair_f16<FMT, true>(y)};
                    k[u] = __builtin_bit_cast(vec<MK, 8>, w);
                    if constexpr (FMT == RL_I8) k[u] -= (MK)KEY_BIAS;
                } else {
                    k[u] = __builtin_bit_cast(vec<MK, 8>, kr[u][st]);
                    // Queries are zeros past the head's end; 16-bit keys may hold what a zero does not cancel.
                    if (a.cache.dim != HD && st * 64 + quad * 16 >= dim_bytes) k[u] = vec<MK, 8>{};
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int p = 0; p < QP; p++) {
                    vec<MK, 8> q;
                    if constexpr (Q_REGS) q = qf[rt][p][st];
                    else q = q_fragment(rt, p, st);
#pragma unroll
                    for (int u = 0; u < 2; u++) S[rt][u] = mfma(k[u], q, S[rt][u]);
                }
        }
        const f32x4 step[2] = {ks[0], ks[1]};
        Place next{{0, 0}};
        if constexpr (MORE) {
            const int32_t t1 = t0 + (int)(ATTEND_WAVES * ATTEND_TILE);
            next = place(t1, ahead);
            ahead = fetch((int32_t)(t1 + ATTEND_WAVES * ATTEND_TILE));
            __builtin_amdgcn_sched_barrier(0);
            load_keys(next);
            __builtin_amdgcn_sched_barrier(0);
        }
        // A tile that some row of the block does not see all of.
        const bool edge = t0 < begin_max || end_min - t0 < (int)ATTEND_TILE;
        vec<MV, 8> w[RT][PP];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            float x[8], most = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if constexpr (EIGHT) x[j] = S[rt][j / 4][j % 4] * (step[j / 4][j % 4] * mult[rt]);
                else x[j] = S[rt][j / 4][j % 4] * mult[rt];
                if (edge) {
                    const int32_t t = t0 + j / 4 * 16 + (int)quad * 4 + j % 4;
                    if (t < row_begin[rt] || t >= row_end[rt]) x[j] = -INFINITY;
                }
                most = fmaxf(most, x[j]);
            }
            most = fmaxf(rows_max(most), top[rt]);
            if (__any(most > top[rt])) {
                const float keep = most == -INFINITY ? 1.0f : exp2_fast(top[rt] - most);
                total[rt] *= keep;
#pragma unroll
                for (int m = 0; m < VD; m++) O[rt][m] *= keep;
                top[rt] = most;
            }
            const float base = (most == -INFINITY ? 0.0f : most) - LIFT;
            float rest[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float p = exp2_fast(x[j] - base);
                total[rt] += p;
                if constexpr (EIGHT) {
                    p *= vs[j / 4][j % 4];
                    if (edge && x[j] == -INFINITY) p = 0.0f; // whatever the step of an unseen token is
                }
                rest[j] = p;
            }
            if constexpr (std::is_same_v<MV, bhalf_t>) { // the first part cut off, not rounded: a mask, and one v_perm for two
                u32x4 cut;
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const uint32_t u0 = __float_as_uint(rest[j]), u1 = __float_as_uint(rest[j + 1]);
                    cut[j / 2] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
                    rest[j] -= __uint_as_float(u0 & 0xFFFF0000u);
                    rest[j + 1] -= __uint_as_float(u1 & 0xFFFF0000u);
                }
                w[rt][0] = __builtin_bit_cast(vec<MV, 8>, cut);
            } else
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    w[rt][0][j] = (MV)rest[j];
                    rest[j] -= (float)w[rt][0][j];
                }
#pragma unroll
            for (int i = 1; i < PP; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    w[rt][i][j] = (MV)rest[j];
                    rest[j] -= (float)w[rt][i][j];
                }
        }
        bool stray = false;
        constexpr uint32_t E = std::is_same_v<MV, half_t> ? 0x7C00u : 0x7F80u; // the exponent of what is not finite
        if constexpr (!EIGHT) {
            if (edge) { // values that no row sees may be anything: zeros; one that is not finite may only reach the rows that see it
                uint32_t odd = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int32_t t = t0 + j / 4 * 16 + (int)quad * 4 + j % 4;
                    const bool out = t < begin_min || t >= end_max;
#pragma unroll
                    for (int c = 0; c < VW; c++) {
                        if (out) vr[j][c] = 0;
                        odd |= (vr[j][c] & E) == E || (vr[j][c] >> 16 & E) == E;
                    }
                }
                stray = mixed && __any(odd);
            }
        }
        if (__builtin_expect(stray, 0)) {
            // Such values take part as zeros, and a second product counts those that a row sees: NaN where it sees any.
            vec<MV, 8> sees[RT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int32_t t = t0 + j / 4 * 16 + (int)quad * 4 + j % 4;
                    sees[rt][j] = (MV)(t >= row_begin[rt] && t < row_end[rt] ? 1.0f : 0.0f);
                }
            each_column([&](const u32x4 &v, int column) {
                constexpr uint32_t ONE = std::is_same_v<MV, half_t> ? 0x3C00u : 0x3F80u;
                u32x4 fine, odd;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t m = ((v[j] & E) == E ? 0xFFFFu : 0u) | ((v[j] >> 16 & E) == E ? 0xFFFF0000u : 0u);
                    fine[j] = v[j] & ~m, odd[j] = m & (ONE | ONE << 16);
                }
                multiply(fine, w, column);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    const f32x4 seen = mfma(__builtin_bit_cast(vec<MV, 8>, odd), sees[rt], f32x4{0, 0, 0, 0});
#pragma unroll
                    for (int i = 0; i < 4; i++) O[rt][column][i] = seen[i] > 0.0f ? NAN : O[rt][column][i];
                }
            });
        } else
            each_column([&](const u32x4 &v, int column) { multiply(v, w, column); });
        if constexpr (MORE) {
            __builtin_amdgcn_sched_barrier(0);
            load_values(next);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (; tile + (int)ATTEND_WAVES < part_end; tile += ATTEND_WAVES) step(std::true_type{});
    if (tile < part_end) step(std::false_type{});

#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        total[rt] = rows_sum(total[rt]);
        if (__any(poison)) total[rt] = NAN;
        if (quad == 0) maxima[wave][rt * 16 + col] = top[rt], sums[wave][rt * 16 + col] = total[rt];
    }
    // Every wave's 16 rows side by side in LDS, then each thread adds four columns of a row.
    float *ob = (float *)lds; // [wave][16][HD + 4]
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int m = 0; m < VD; m += 4)
                *(f32x4 *)(ob + (wave * 16 + col) * (HD + 4) + (quad * 4 + i) * VD + m) =
                    f32x4{O[rt][m][i], O[rt][m + 1][i], O[rt][m + 2][i], O[rt][m + 3][i]};
        __syncthreads();
        for (uint32_t i = tid; i < 16 * (HD / 4); i += ATTEND_THREADS) {
            const uint32_t r = rt * 16 + i / (HD / 4), d = i % (HD / 4) * 4;
            if (r >= count) break;
            const uint2 e = by_group(r0 + r);
            float2 ms = make_float2(maxima[0][r], 0.0f);
#pragma unroll
            for (uint32_t v = 1; v < ATTEND_WAVES; v++) ms.x = fmaxf(ms.x, maxima[v][r]);
            f32x4 x = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t v = 0; v < ATTEND_WAVES; v++) { // a wave without tokens adds zeros (or NaN)
                const float f = maxima[v][r] == -INFINITY ? 1.0f : exp2_fast(maxima[v][r] - ms.x);
                ms.y += sums[v][r] * f;
                x += *(const f32x4 *)(ob + (v * 16 + i / (HD / 4)) * (HD + 4) + d) * f;
            }
            const uint64_t row = first + e.x, qh = head * G + e.y, at = row * a.q_heads + qh;
            bool none = span.end(e.x) <= span.begin(e.x);
            if constexpr (MODE != ATTEND_ALONE)
                if (!none && ms.x == -INFINITY) ms.x = ATTEND_LOWEST;
            if constexpr (MODE == ATTEND_PREFIX) {
                const uint64_t slot = at * a.stride + a.shared + part;
                *(f32x4 *)(a.part_out + slot * HD + d) = x;
                if (d == 0) a.part_sum[slot] = ms;
                continue;
            } else if constexpr (MODE == ATTEND_JOINED) {
                if (a.joins) {
                    const uint64_t slot = at * a.stride + a.shared;
                    constexpr uint32_t AHEAD = 8; // parts loaded at a time
                    for (uint32_t p0 = 0; p0 < shared_parts; p0 += AHEAD) {
                        float2 more[AHEAD];
                        f32x4 y[AHEAD];
#pragma unroll
                        for (uint32_t p = 0; p < AHEAD; p++) {
                            const uint64_t from = slot + min(p0 + p, shared_parts - 1);
                            more[p] = a.part_sum[from], y[p] = *(const f32x4 *)(a.part_out + from * HD + d);
                        }
#pragma unroll
                        for (uint32_t p = 0; p < AHEAD; p++)
                            if (p0 + p < shared_parts) attend_add(ms, x, more[p], y[p]);
                    }
                    attend_write<T>(a, row, qh, d, ms.x == -INFINITY, ms, x, LIFT);
                } else {
                    *(f32x4 *)(a.part_out + (at * a.stride + part) * HD + d) = x;
                    if (d == 0) a.part_sum[at * a.stride + part] = ms;
                    if (d == 0 && part == 0) a.part_count[at] = parts | (shared_parts ? 0 : ATTEND_NONE);
                }
                continue;
            }
            if (parts == 1) attend_write<T>(a, row, qh, d, none, ms, x, LIFT);
            else if (a.joins) {
                shared_store(a.part_out + (at * a.parts + part) * HD + d, float2{x[0], x[1]});
                shared_store(a.part_out + (at * a.parts + part) * HD + d + 2, float2{x[2], x[3]});
                if (d == 0) shared_store((float *)(a.part_sum + at * a.parts + part), ms);
            } else {
                *(f32x4 *)(a.part_out + (at * a.parts + part) * HD + d) = x;
                if (d == 0) a.part_sum[at * a.parts + part] = ms;
                if (d == 0 && part == 0) a.part_count[at] = parts | (none ? ATTEND_NONE : 0);
            }
        }
    }
    if (MODE != ATTEND_ALONE || parts == 1 || !a.joins) return;
    // The last of the block's parts to arrive joins them. Every wave's results are written before the arrival, and both
    // sides go past the caches that XCDs do not share.
    __builtin_amdgcn_s_waitcnt(ATTEND_STORED);
    __syncthreads();
    const auto of = [&](uint32_t r) {
        const uint2 e = by_group(r0 + r);
        return (uint64_t)(first + e.x) * a.q_heads + head * G + e.y;
    };
    if (tid == 0) {
        uint32_t *arrived = a.arrived + of(0);
        last = atomicAdd(arrived, 1u) == parts - 1;
        if (last) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); // ready for the next call
    }
    __syncthreads();
    if (!last) return;
    float *factor = (float *)lds; // [ROWS][ATTEND_FEW]
    {
        constexpr uint32_t EACH = ATTEND_FEW / TPR;
        const uint32_t j = tid % TPR;
        const float2 *sum_of = a.part_sum + of(q_row < count ? q_row : 0) * a.parts;
        float2 ms[EACH];
        float most = -INFINITY, sum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < EACH; i++) {
            const uint32_t p = j + i * TPR;
            ms[i] = shared_load((const float *)(sum_of + (p < parts ? p : 0)));
            if (p >= parts) ms[i] = make_float2(-INFINITY, 0.0f);
            most = fmaxf(most, ms[i].x);
        }
        most = group_max<TPR>(most);
#pragma unroll
        for (uint32_t i = 0; i < EACH; i++) {
            const float f = ms[i].x == -INFINITY ? 0.0f : exp2_fast(ms[i].x - most);
            factor[q_row * ATTEND_FEW + j + i * TPR] = f;
            sum += ms[i].x == -INFINITY ? ms[i].y : ms[i].y * f; // a part without tokens has 0, or NaN
        }
        sum = group_sum<TPR>(sum);
        if (j == 0) maxima[0][q_row] = most, sums[0][q_row] = sum;
    }
    __syncthreads();
    for (uint32_t i = tid; i < count * (HD / 4); i += ATTEND_THREADS) {
        const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4;
        const uint2 e = by_group(r0 + r);
        const float *x = a.part_out + of(r) * a.parts * HD + d;
        f32x4 all = {0, 0, 0, 0};
        for (uint32_t p0 = 0; p0 < parts; p0 += 8) {
            float2 y[8][2];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                const float *z = x + (p0 + j < parts ? p0 + j : p0) * HD;
                y[j][0] = shared_load(z), y[j][1] = shared_load(z + 2);
            }
#pragma unroll
            for (uint32_t j = 0; j < 8; j++)
                if (p0 + j < parts) all += f32x4{y[j][0].x, y[j][0].y, y[j][1].x, y[j][1].y} * factor[r * ATTEND_FEW + p0 + j];
        }
        attend_write<T>(a, first + e.x, head * G + e.y, d, span.end(e.x) <= span.begin(e.x),
                        make_float2(maxima[0][r], sums[0][r]), all, LIFT);
    }
