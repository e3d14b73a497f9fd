// bw_attention_body.h - the body of the attention kernels in bw_attention_kernel.h: template parameters F and FOLD, argument a, and WINDOW, whether only the tokens of a
// window and the sinks count.  (Included by both rather than called: a function that is given the kernel's arguments holds them in registers from the start, and
// the kernels that use them all spill 50 ... 70 bytes more.)
    constexpr int kChunk = F::kDim < 128 ? F::kDim : 128, kPitch = kChunk + 4, kChunkBlocks = kChunk / 16;
    __shared__ float outs[kWaves][kQueries][kPitch];
    __shared__ float stats[kWaves][2][kQueries];
    __shared__ uint32_t lds[8];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), m = lane & 15, kg = lane >> 4;
    using Z = Fold<FOLD>;
    const Z fold(m);
    const int column = m & (Z::kColumns - 1);
    const Exchange<F::kMerge> exchanged(m);
    const uint32_t per_seq = (uint32_t)(a.kv_heads * a.q_groups);

    // the piece of this workgroup: from unit `at` of segment (b, hq) on, `left` units in all
    uint32_t b, hq, at, left;
    Split s = {};
    if (a.whole) {
        b = blockIdx.x / per_seq;
        hq = blockIdx.x - b * per_seq;
        at = 0;
        left = visible_of<WINDOW>(a, tokens_of(a, b)).tiles + kSegmentCost;
    } else {
        const Place place = find_sequence<WINDOW>(a, lds, [&](uint32_t all, uint32_t before, uint32_t units) {
            s = split_of(a, all, gridDim.x);
            const uint32_t start = s.start(blockIdx.x);
            return blockIdx.x < s.pieces && before * per_seq <= start && start < (before + units) * per_seq;
        });
        if (threadIdx.x == 0) a.joints[blockIdx.x].parts = 0;
        for (uint32_t e = blockIdx.x; e < (uint32_t)a.B; e += gridDim.x) {      // sequences without tokens
            if (tokens_of(a, e) > 0) continue;
            uint2* out = reinterpret_cast<uint2*>(a.out + (int64_t)e * a.q_heads * a.dim);
            for (int i = (int)threadIdx.x; i < a.q_heads * a.dim / 4; i += 256) out[i] = uint2{0, 0};
        }
        s = split_of(a, place.all, gridDim.x);
        if (blockIdx.x >= s.pieces) return;
        const uint32_t start = s.start(blockIdx.x), rest = start - place.before * per_seq;
        left = s.start(blockIdx.x + 1) - start;
        b = place.b;
        const uint32_t units = units_of<WINDOW>(a, tokens_of(a, b));
        hq = rest / units;
        at = rest - hq * units;
    }
    Segment g = segment_of<WINDOW>(a, b, hq, at, left);
    if (g.from >= g.to && !a.whole) return;
    uint32_t position = s.start(blockIdx.x);                      // of the segment's units of this piece, among all (not of whole segments)
    const int page_mask = (1 << a.page_shift) - 1;

    // ---- addresses ----
    uint32_t key_off[F::kCodes ? F::kGroups : F::NK], value_off[F::kValueLoads];
    if constexpr (F::kCodes) {
#pragma unroll
        for (int c = 0; c < F::kGroups; c++) key_off[c] = (uint32_t)(m * a.row_bytes + (c * F::kGroup + kg * (F::kGroup / 4)) * F::kBits / 8);
#pragma unroll
        for (int w = 0; w < F::kMerged; w++)
            value_off[w] = (uint32_t)(4 * kg * a.row_bytes + (w * F::kMerge + m % F::kMerge) * F::kGroupBytes + m / F::kMerge * (F::kMerge * F::kValueBytes));
#pragma unroll
        for (int w = F::kMerged; w < F::kValueLoads; w++)
            value_off[w] = (uint32_t)(4 * kg * a.row_bytes + (F::kMerged * (F::kMerge - 1) + w) * F::kGroupBytes + m * F::kValueBytes);
    } else {
#pragma unroll
        for (int k = 0; k < F::NK; k++) key_off[k] = (uint32_t)(m * a.row_bytes + (F::k_at(k, kg) < a.dim ? 2 * F::k_at(k, kg) : 0));
#pragma unroll
        for (int h = 0; h < F::kValueLoads; h++) value_off[h] = (uint32_t)(4 * kg * a.row_bytes + (F::v_at(m, 8 * h) < a.dim ? 2 * F::v_at(m, 8 * h) : 0));
    }
    constexpr int kAhead = tiles_ahead<F, FOLD>;
    Tile<F> ring[kAhead];                                         // the ones under way: asked for, or worked on
    u4 q_raw[F::NK];
    auto halves_of = [&](const Segment& g, uint32_t t) {         // (one of which no token counts has no page, whatever the table says)
        const int at = (int)t * kTile;
        Halves h;
        h.page[0] = !WINDOW || at + 16 > g.seen.from || at < a.sinks ? (uint32_t)uniform_load(g.table, at >> a.page_shift) : 0xFFFFFFFFu;
        h.page[1] = at + 16 < g.n && (!WINDOW || at + 32 > g.seen.from || at + 16 < a.sinks) ? (uint32_t)uniform_load(g.table, (at + 16) >> a.page_shift) : 0xFFFFFFFFu;
        return h;
    };
    auto row_of = [&](const Segment& g, const Halves& h, uint32_t t, int half) {  // row of the half's first token, in rows of this head's pages
        const uint32_t page = h.page[half] < a.pages ? h.page[half] : 0;
        return (((int64_t)page * a.kv_heads + g.head) << a.page_shift) + (((int)t * kTile + 16 * half) & page_mask);
    };
    // where the lane's pairs lie (FOLD 2: the keys'; the values' lie as far from value_meta)
    const int pair_token = fold.pair_token(m);
    const uint32_t* pair_base = (FOLD != 2 && Z::pair_is_value(m) ? a.value_meta : a.key_meta) + 4 * kg + (pair_token & 3);
    auto load_keys = [&](Tile<F>& tile, const Segment& g, uint32_t t) __attribute__((always_inline)) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint8_t* base = a.keys + row_of(g, tile.h, t, half) * a.row_bytes;
            if constexpr (F::kCodes) {
#pragma unroll
                for (int c = 0; c < F::kGroups; c++) load_words<F::kKeyGroupWords>(base + key_off[c], tile.key[half] + c * F::kKeyGroupWords);
            } else {
#pragma unroll
                for (int k = 0; k < F::NK; k++) load_words<4>(base + key_off[k], tile.key[half] + 4 * k);
            }
        }
        if constexpr (F::kCodes) {
            int64_t at[2];
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint32_t page = tile.h.page[half] < a.pages ? tile.h.page[half] : 0;
                at[half] = ((((int64_t)page * a.kv_heads + g.head) * F::kGroups) << a.page_shift) + (((int)t * kTile + 16 * half) & page_mask);
            }
            const uint32_t* p = pair_base + (pair_token & 4 ? at[1] : at[0]);
#pragma unroll
            for (int c = 0; c < F::kGroups; c++) {
                tile.pairs[0][c] = p[c << a.page_shift];
                if constexpr (FOLD == 2) tile.pairs[1][c] = (a.value_meta - a.key_meta + p)[c << a.page_shift];
            }
        }
    };
    auto load_values = [&](Tile<F>& tile, const Segment& g, uint32_t t) __attribute__((always_inline)) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint8_t* base = a.values + row_of(g, tile.h, t, half) * a.row_bytes;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint8_t* row = base + i * a.row_bytes;
                uint32_t* out = tile.value[4 * half + i];
                if constexpr (F::kCodes) {
#pragma unroll
                    for (int w = 0; w < F::kMerged; w++)
                        load_words<F::kValueGroupWords, kPast<F>>(row + value_off[w], out + w * F::kValueGroupWords);
#pragma unroll
                    for (int w = F::kMerged; w < F::kValueLoads; w++) {
                        if constexpr (F::kValueBytes == 2) out[w] = *reinterpret_cast<const uint16_t*>(row + value_off[w]);
                        else out[w] = row[value_off[w]];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < F::kValueLoads; k++) load_words<F::kDim == 64 ? 2 : 4, kPast<F>>(row + value_off[k], out + 4 * k);
                }
            }
        }
    };
    // A segment's queries and first tiles: asked for while the segment before it is put together.
    auto begin = [&](const Segment& g) __attribute__((always_inline)) {
        const uint16_t* src = a.q + g.b * a.q_row + (g.q_head + (column < g.queries ? column : 0)) * a.q_head;
#pragma unroll
        for (int k = 0; k < F::NK; k++) {
            const int d = F::k_at(k, kg);
            q_raw[k] = column < g.queries && d < a.dim ? *reinterpret_cast<const u4*>(src + d) : u4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (g.from + wave + i * kWaves >= g.to) break;
            const uint32_t nth = g.from + wave + i * kWaves, t = WINDOW ? g.place(nth) : nth;
            ring[i].h = halves_of(g, t);
            load_keys(ring[i], g, t);
            load_values(ring[i], g, t);
        }
    };
    begin(g);
    for (;;) {
        left -= g.units;
        Segment after = g;
        bool more_segments = false;
        if (left) {
            if (++hq == per_seq) {
                hq = 0;
                do
                    if (++b >= (uint32_t)a.B) return;             // (never, while nobody writes the lengths)
                while (tokens_of(a, b) == 0);
            }
            after = segment_of<WINDOW>(a, b, hq, 0, left);
            more_segments = after.from < after.to;
        }
        const int n = g.n;
        const uint32_t to = g.to;

        // ---- Q: over codes brought near 2^14 by a power of two, with the sum of every group in the codes' unit ----
        float q_sum[F::kGroups], score_scale = a.scale;
        u4 q[F::NK];
#pragma unroll
        for (int k = 0; k < F::NK; k++) q[k] = q_raw[k];
        if constexpr (F::kCodes) {
            float x[F::NK][8], top = 0.f;
#pragma unroll
            for (int k = 0; k < F::NK; k++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint16_t u = (uint16_t)(q[k][e / 2] >> (16 * (e & 1)));
                    x[k][e] = a.q_bf16 ? bf16_to_f32(u) : f16_bits(u);
                    top = fmaxf(top, __builtin_fabsf(x[k][e]));
                }
            // exact but for values 2^28 and more below the largest
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const int ex = top > 0.f && top <= 3.4e38f ? __builtin_amdgcn_frexp_expf(top) - 14 : 0;
            score_scale = __builtin_ldexpf(a.scale, ex + kUnit<F::kBits>);
            // (queries beyond 2^120: the largest number keeps scores finite that are, and they are 2^100 apart either way)
            if (__builtin_isinf(score_scale)) score_scale = __builtin_copysignf(3.4028235e38f, score_scale);
#pragma unroll
            for (int c = 0; c < F::kGroups; c++) {
                float sum = 0.f;
#pragma unroll
                for (int k = c * F::kPerK; k < (c + 1) * F::kPerK; k++) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[k][e] = __builtin_ldexpf(x[k][e], -ex);
                        sum += x[k][e];
                    }
#pragma unroll
                    for (int p = 0; p < 4; p++)
                        q[k][p] = as_u32(h2{(_Float16)x[k][query_order<F::kBits>(2 * p)], (_Float16)x[k][query_order<F::kBits>(2 * p + 1)]});
                }
                sum += __shfl_xor(sum, 16, 64);
                q_sum[c] = __builtin_ldexpf(sum + __shfl_xor(sum, 32, 64), -kUnit<F::kBits>);
            }
        }

        // ---- tiles ----
        f4 acc[F::NV], zeros[F::kGroups];                         // zeros: sums of (P s) z, the same in every row
        float r = kLowest, l = 0.f, reach[F::kGroups];
        bool any = false;                                         // a token that counts, for any lane
#pragma unroll
        for (int j = 0; j < F::NV; j++) acc[j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < F::kGroups; c++) {
            zeros[c] = f4{0.f, 0.f, 0.f, 0.f};
            reach[c] = __builtin_ldexpf(1.f, kFirstReach);
        }
        auto step = [&](Tile<F>& tile, const uint32_t nth) __attribute__((always_inline)) {
            // The second half of the workgroups shares its CUs with the first, whose waves, being older, go before: 17 against 21 us of a launch's 24.
            // Going first every other tile evens it out (48 sequences of up to 8192 tokens, 8 heads of 128 in 8 bits: 46.2 against 47.4 us).
            __builtin_amdgcn_s_setprio(0);
            if (blockIdx.x >= gridDim.x / 2 && (nth / kWaves & 1)) __builtin_amdgcn_s_setprio(1);
            const uint32_t t = WINDOW ? g.place(nth) : nth, next = WINDOW ? g.place(nth + kAhead * kWaves) : nth + kAhead * kWaves;
            const bool more = nth + kAhead * kWaves < to;
            Halves hn = {};
            if (more) hn = halves_of(g, next);
            // Tokens that do not count: behind the end, before the window and no sink, or on a page outside the cache.
            const bool full = (int)t * kTile + kTile <= n && (!WINDOW || (int)t * kTile >= g.seen.from || (int)t * kTile + kTile <= a.sinks) && tile.h.page[0] < a.pages && tile.h.page[1] < a.pages;
            const Halves h = tile.h;
            any |= h.page[0] < a.pages || h.page[1] < a.pages;
            auto counts = [&](int half, int i) {
                const int token = (int)t * kTile + 16 * half + 4 * kg + i;
                return token < n && (!WINDOW || token >= g.seen.from || token < a.sinks) && h.page[half] < a.pages;
            };
            auto seen = [&](int e) { return counts(e >> 2, e & 3); };               // of the lane's 8 tokens
            auto own = [&](int j) { const int e = fold.token(j); return e & 4 ? counts(1, e & 3) : counts(0, e & 3); };
            uint32_t pairs[2][F::kGroups];
            if constexpr (F::kCodes) {
#pragma unroll
                for (int c = 0; c < F::kGroups; c++)
#pragma unroll
                    for (int w = 0; w < Z::kRegisters; w++) pairs[w][c] = tile.pairs[w][c];
                if (!full) {
                    const bool counted = pair_token & 4 ? counts(1, pair_token & 3) : counts(0, pair_token & 3);
#pragma unroll
                    for (int c = 0; c < F::kGroups; c++)
#pragma unroll
                        for (int w = 0; w < Z::kRegisters; w++) pairs[w][c] = counted ? pairs[w][c] : 0u;
                }
            }
            // scores, in units of log 2
            float x[Z::kTokens];
            if constexpr (F::kCodes) {
#pragma unroll
                for (int c = 0; c < F::kGroups; c++) {
                    f4 dot[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        uint32_t codes[4 * F::kPerK];
#pragma unroll
                        for (int w = 0; w < F::kKeyGroupWords; w++) key_codes<F::kBits>(tile.key[half][c * F::kKeyGroupWords + w], codes + w * (16 / F::kBits));
#pragma unroll
                        for (int k = 0; k < F::kPerK; k++)
                            dot[half] = mfma<false>(u4{codes[4 * k], codes[4 * k + 1], codes[4 * k + 2], codes[4 * k + 3]}, q[c * F::kPerK + k], dot[half]);
                    }
                    const uint32_t zero = pairs[0][c] >> 16;
                    static_for<0, Z::kTokens>([&](auto jc) {
                        constexpr int j = decltype(jc)::value;
                        const float part = __builtin_fmaf(-f16_bits(Z::template key_pair<j>(zero)), q_sum[c], fold.template pick<j>(dot));
                        const float scale = f16_bits(Z::template key_pair<j>(pairs[0][c]));
                        x[j] = c ? __builtin_fmaf(scale, part, x[j]) : scale * part;
                    });
                }
            } else {
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < F::NK; k++) {
                        const uint32_t* w = tile.key[half] + 4 * k;
                        s = mfma<F::kBf16>(u4{w[0], w[1], w[2], w[3]}, q[k], s);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) x[4 * half + i] = s[i] * score_scale;
                }
            }
            if (more) {
                tile.h = hn;
                load_keys(tile, g, next);
            }
            if constexpr (F::kCodes) {
#pragma unroll
                for (int j = 0; j < Z::kTokens; j++) x[j] *= score_scale;
            }
            if (!full) {
#pragma unroll
                for (int j = 0; j < Z::kTokens; j++) x[j] = own(j) ? x[j] : -INFINITY;
            }
            auto over_lanes = [&](float top) {                   // of a query's column
                top = Z::max(top);
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                return fmaxf(top, __shfl_xor(top, 32, 64));
            };
            float top = x[0];
#pragma unroll
            for (int j = 1; j < Z::kTokens; j++) top = fmaxf(top, x[j]);
            const bool passed = __builtin_amdgcn_ballot_w64(top > r + (F::kCodes ? kSlack : kMost<F::kBf16>));
            float raise = 0.f;                                    // of r, over codes
            if (passed) {
                top = over_lanes(top);
                if constexpr (F::kCodes) {
                    const float raised = fmaxf(top, r);
                    raise = raised == r ? 0.f : fminf(raised - r, 300.f);
                    r = raised;
                    l *= __builtin_amdgcn_exp2f(-raise);
                } else {
                    const float raised = fmaxf(top - kTop<F::kBf16>, r), keep = raised == r ? 1.f : __builtin_amdgcn_exp2f(r - raised);
                    r = raised;
                    l *= keep;
#pragma unroll
                    for (int j = 0; j < F::NV; j++) acc[j] *= keep;
                }
            }
            float p[Z::kTokens];
#pragma unroll
            for (int j = 0; j < Z::kTokens; j++) p[j] = __builtin_amdgcn_exp2f(x[j] - r);       // (r is never minus infinity: 0 where x is)
#pragma unroll
            for (int j = 0; j < Z::kTokens; j++) l += p[j];
            // weighted values
            if constexpr (F::kCodes) {
                if constexpr (F::kMerge > 1) {
#pragma unroll
                    for (int w = 0; w < F::kMerged; w++)
#pragma unroll
                        for (int e = 0; e < 8; e++) tile.value[e][w] = exchanged(tile.value[e][w]);
                }
                static_for<0, F::kGroups>([&](auto cc) {
                    constexpr int c = decltype(cc)::value;
                    float ps[Z::kTokens], most = 0.f;             // P s, times the group's reach
                    static_for<0, Z::kTokens>([&](auto jc) {
                        constexpr int j = decltype(jc)::value;
                        ps[j] = p[j] * f16_bits(Z::template value_pair<j>(pairs[0][c], pairs[Z::kRegisters - 1][c])) * reach[c];
                        most = fmaxf(most, __builtin_fabsf(ps[j]));
                    });
                    if (passed || __builtin_amdgcn_ballot_w64(most > (float)(1 << kMost<false>))) {
                        most = over_lanes(most);
                        // up with the reference (by whole powers of two; what they are more goes into the sums), so that the group's weights do not
                        // sink; down where they would pass 2^kMost
                        const int up = (int)__builtin_ceilf(raise);
                        const int was = __builtin_amdgcn_frexp_expf(reach[c]) - 1, high = most > 0.f ? __builtin_amdgcn_frexp_expf(most) - was : -1000;
                        int now = min(was + up, kFirstReach);
                        if (high + now > kMost<false>) now = min(kTop<false> + 1 - high, now);
                        reach[c] = __builtin_ldexpf(1.f, now);
#pragma unroll
                        for (int j = 0; j < Z::kTokens; j++) ps[j] = __builtin_ldexpf(ps[j], now - was);
                        const float by = __builtin_ldexpf(__builtin_amdgcn_exp2f((float)up - raise), now - was - up);
#pragma unroll
                        for (int j = 0; j < F::kPerV; j++) acc[c * F::kPerV + j] *= by;
                        zeros[c] *= by;
                    }
                    uint32_t own_hi[Z::kTokens / 2], own_lo[Z::kTokens / 2];
#pragma unroll
                    for (int i = 0; i < Z::kTokens / 2; i++) {
                        own_hi[i] = split_pair<false>(ps[2 * i], ps[2 * i + 1]);
                        own_lo[i] = pair_of<false>(ps[2 * i], ps[2 * i + 1]);
                    }
                    const u4 hi = Z::all(own_hi), lo = Z::all(own_lo);
                    const uint32_t pair = pairs[Z::kRegisters - 1][c], both = token_pair<true>((uint32_t)__builtin_amdgcn_mov_dpp((int)pair, 0xB1, 0xF, 0xF, true), pair);
                    u4 z;
                    static_for<0, 4>([&](auto ic) { z[decltype(ic)::value] = Z::template zero_pair<decltype(ic)::value>(both); });
                    u4 v[F::kPerV];
                    static_for<0, F::kPerV>([&](auto jc) {
                        constexpr int j = decltype(jc)::value, w = F::value_word(c, j);
#pragma unroll
                        for (int i = 0; i < 4; i++) v[j][i] = value_codes<F::kBits, F::value_code(c, j)>(tile.value[2 * i + 1][w], tile.value[2 * i][w]);
                        acc[c * F::kPerV + j] = mfma<false>(v[j], hi, acc[c * F::kPerV + j]);
                    });
                    zeros[c] = mfma<false>(z, hi, zeros[c]);
#pragma unroll
                    for (int j = 0; j < F::kPerV; j++) acc[c * F::kPerV + j] = mfma<false>(v[j], lo, acc[c * F::kPerV + j]);
                    zeros[c] = mfma<false>(z, lo, zeros[c]);
                });
            } else {
                if (!full) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
#pragma unroll
                        for (int w = 0; w < F::kValueWords; w++) tile.value[e][w] = seen(e) ? tile.value[e][w] : 0u;
                }
                constexpr int kParts = F::kBf16 ? 3 : 2;
                u4 part[kParts];
#pragma unroll
                for (int i = 0; i < 4; i++) {
#pragma unroll
                    for (int n = 0; n < kParts - 1; n++) part[n][i] = split_pair<F::kBf16>(p[2 * i], p[2 * i + 1]);
                    part[kParts - 1][i] = pair_of<F::kBf16>(p[2 * i], p[2 * i + 1]);
                }
                static_for<0, F::NV>([&](auto jc) {
                    constexpr int j = decltype(jc)::value;
                    u4 v;
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = token_pair<(j & 1) != 0>(tile.value[2 * i + 1][j / 2], tile.value[2 * i][j / 2]);
#pragma unroll
                    for (int n = 0; n < kParts; n++) acc[j] = mfma<F::kBf16>(v, part[n], acc[j]);
                });
            }
            if (more) load_values(tile, g, next);
        };
        for (uint32_t t = g.from + wave; t < to; t += kAhead * kWaves) {
            step(ring[0], t);
            if constexpr (kAhead == 2)
                if (t + kWaves < to) step(ring[1], t + kWaves);
        }
        if (more_segments) begin(after);

        // ---- the four waves of the workgroup joined ----
        if (!any) r = -INFINITY;
        l = Z::sum(l);
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (lane < Z::kColumns) {
            stats[wave][0][m] = r;
            stats[wave][1][m] = l;
        }
        __syncthreads();
        const float r_all = fmaxf(fmaxf(stats[0][0][column], stats[1][0][column]), fmaxf(stats[2][0][column], stats[3][0][column]));
        const float f = r == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r - r_all);
        const bool complete = g.from == 0 && to == g.tiles;
        float* slot = complete ? nullptr : a.partial + (int64_t)(2 * blockIdx.x + (g.from == 0)) * (2 * kQueries + a.queries * a.dim);
        if (!complete && g.from == 0 && threadIdx.x == 0)         // (the segment ends tiles - to units behind this piece)
            a.joints[blockIdx.x] = Joint{g.b, g.hq, min(s.piece_of(position + g.units + g.tiles - to - 1), s.pieces - 1) - blockIdx.x + 1};
        auto joined = [&](int query, float& top) {                // sum of the waves' l, relative to the largest r
            top = fmaxf(fmaxf(stats[0][0][query], stats[1][0][query]), fmaxf(stats[2][0][query], stats[3][0][query]));
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                const float rw = stats[w][0][query];
                sum += (rw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(rw - top)) * stats[w][1][query];
            }
            return sum;
        };
        const int queries = g.queries;
        if (!complete && threadIdx.x < (uint32_t)queries) {
            float top;
            slot[kQueries + threadIdx.x] = joined((int)threadIdx.x, top);
            slot[threadIdx.x] = top;
        }
#pragma unroll
        for (int c = 0; c < (F::NV + kChunkBlocks - 1) / kChunkBlocks; c++) {
            if (c) __syncthreads();
            if (m < queries) {
#pragma unroll
                for (int j = c * kChunkBlocks; j < (c + 1) * kChunkBlocks && j < F::NV; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float o = acc[j][i];
                        if constexpr (F::kCodes)
                            o = __builtin_ldexpf(__builtin_fmaf(o, (float)(1 << kUnit<F::kBits>), -zeros[j / F::kPerV][i]), 1 - __builtin_amdgcn_frexp_expf(reach[j / F::kPerV]));
                        outs[wave][m][F::v_at(4 * kg + i, j) - c * kChunk] = o * f;
                    }
            }
            __syncthreads();
            for (int e = (int)threadIdx.x; e < queries * (kChunk / 4); e += 256) {
                const int query = e / (kChunk / 4), d = (e - query * (kChunk / 4)) * 4;
                if (c * kChunk + d >= a.dim) continue;
                f4 o = *reinterpret_cast<const f4*>(&outs[0][query][d]);
#pragma unroll
                for (int w = 1; w < kWaves; w++) o += *reinterpret_cast<const f4*>(&outs[w][query][d]);
                if (complete) {
                    float top;
                    const float sum = joined(query, top), inv = top == -INFINITY ? 0.f : 1.f / sum;
                    store_out(a, (int64_t)g.b * a.q_heads + g.q_head + query, c * kChunk + d, o * inv);
                } else {
                    *reinterpret_cast<f4*>(slot + 2 * kQueries + query * a.dim + c * kChunk + d) = o;
                }
            }
        }
        if (!more_segments) break;
        __syncthreads();                                          // (the next segment writes stats and outs again)
        position += g.units;
        g = after;
    }
