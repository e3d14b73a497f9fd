// bw_prompt_grad_kernel.h - gradients of the attention in bw_prompt_kernel.h.  With P = 2^(S c - lse), the weights of the forward again, and g the output's gradient:
//   dP = g V^T,  delta = rowsum(g out),  dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T g
// One kernel has the rows and goes over the keys (dQ, and delta on the way), another has the keys and goes over the rows (dK, dV), so that every sum is one
// workgroup's, in one order, and nothing is added up in memory: seven products where five would do, and the same bits every time.
//
// P and dS enter their second product as 16-bit numbers, rounded once.  In float16, whose steps end at 2^-24, P goes in 2^12 times as large, and dS times a power of two that
// is each row's (each key's) own: it starts high and comes down where a product would pass 2^15, and the sums with it.
#pragma once
#include "bw_prompt_kernel.h"

struct PromptGradArgs {
    PromptArgs p;
    const uint16_t *grad, *result;               // of the output; result [tokens][q_heads][dim]
    int64_t grad_row, grad_head;
    float* delta;                                // as lse
    uint16_t *q_grad, *k_grad, *v_grad;
    float* parts;                                // [splits][k_tokens][kv_heads][2][dim], where splits > 1
    float* sink_parts;                           // [sequences][kv_heads][far][sinks][2][dim]
    int far;                                     // workgroups that share the rows which see a sequence's sinks and not their window; 0: none
    float plain_scale;
};

constexpr int kFirstReach16 = 80, kReachTop = 12, kReachMost = 15, kWeightShift = 12;

// The power of two (of each lane) that its values `x`, times 2^reach, go into a product with, which brings down the sums in `acc` where it comes down.
template <int N, int BLOCKS> BW_DEV void fit_reach(float* x, int& reach, f16v* acc) {
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < N; j++) most = fmaxf(most, __builtin_fabsf(x[j]));
    const float factor = __builtin_ldexpf(1.f, reach);
    if (__builtin_amdgcn_ballot_w64(most * factor > (float)(1 << kReachMost))) {
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        const int high = most > 0.f && most <= 3.4e38f ? __builtin_amdgcn_frexp_expf(most) : -1000;
        const int now = high + reach > kReachMost ? kReachTop + 1 - high : reach;
        const float by = __builtin_ldexpf(1.f, now - reach);
        reach = now;
#pragma unroll
        for (int m = 0; m < BLOCKS; m++) acc[m] *= by;
    }
    const float with = __builtin_ldexpf(1.f, reach);
#pragma unroll
    for (int j = 0; j < N; j++) x[j] *= with;
}

// 16 values of a lane as the second operand of two MFMAs.
template <int DT> BW_DEV void pack16(const float* x, u4* w) {
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) w[t][j] = narrow_pair<DT>(x[8 * t + 2 * j], x[8 * t + 2 * j + 1]);
}

template <class H>
__global__ __launch_bounds__(256, H::kResident) void prompt_query_grad_kernel(PromptGradArgs g) {
    extern __shared__ __align__(1024) char smem[];               // [2][K, V]
    constexpr int DT = H::kType;
    const PromptArgs& a = g.p;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5;
    Span p;
    int head;
    uint32_t split;
    if (!place_of<kRows, false>(a, p, head, split)) return;
    clear_tiles<H>(smem, 4 * H::kTileBytes, a.dim);
    const int row0 = p.tile * kRows + wave * kWaveRows, rows = p.nq * a.share;
    const Row row(a, p, row0 + (lane & 31));
    const int64_t token = p.q0 + row.token, index = (int64_t)head * a.q_tokens * a.share + token * a.share + row.head;
    u4 q[H::kSteps], grad[H::kSteps];
    load_row<H>(q, a.q + token * a.q_row + (head * a.share + row.head) * a.q_head, row.live, a.dim, half);
    load_row<H>(grad, g.grad + token * g.grad_row + (head * a.share + row.head) * g.grad_head, row.live, a.dim, half);
    float delta = 0.f;
    {
        const uint16_t* result = g.result + (token * a.q_heads + head * a.share + row.head) * a.dim;
#pragma unroll
        for (int s = 0; s < H::kSteps; s++) {
            const int d = 16 * s + 8 * half;
            const u4 o = row.live && d < a.dim ? *reinterpret_cast<const u4*>(result + d) : u4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                delta = __builtin_fmaf(widen16<DT>((uint16_t)o[j]), widen16<DT>((uint16_t)grad[s][j]), delta);
                delta = __builtin_fmaf(widen16<DT>((uint16_t)(o[j] >> 16)), widen16<DT>((uint16_t)(grad[s][j] >> 16)), delta);
                q[s][j] ^= a.flip;
            }
        }
        delta += __shfl_xor(delta, 32, 64);
    }
    if (row.live && half == 0) g.delta[index] = delta;
    if (!g.q_grad) return;
    const float lse = row.live ? a.lse[index] : INFINITY;

    int low, high, wave_low, wave_high;
    positions_of(a, p, p.tile * kRows, (p.tile + 1) * kRows, low, high);
    positions_of(a, p, row0 < rows ? row0 : p.tile * kRows, row0 + kWaveRows, wave_low, wave_high);
    const KeyTiles tiles(a, low, high, p.nk, H::kKeys);
    const RowLoader<H> load_k(lane, wave, a.k_row), load_v(lane, wave, a.v_row);
    const TileReader<H> read(lane);
    const uint16_t *keys = a.k + p.k0 * a.k_row + head * a.k_head, *values = a.v + p.k0 * a.v_row + head * a.v_head;
    const uint32_t lds = lds_address(smem);
    auto fetch = [&](int i) __attribute__((always_inline)) {
        const int64_t at = (int64_t)tiles[i] * H::kKeys;
        const int n = p.nk - (int)at;
        const uint32_t to = lds + (i & 1) * 2 * H::kTileBytes;
        load_k(keys + at * a.k_row, n, to, wave, a.dim);
        load_v(values + at * a.v_row, n, to + H::kTileBytes, wave, a.dim);
    };

    f16v acc[H::kBlocks];
    int reach = 0;
    for (int careful = 0;; careful = 1) {                        // (see prompt_forward_kernel)
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++) acc[m] = f16v{};
        reach = kFirstReach16;
        if (tiles.count) fetch(0);
        for (int i = 0; i < tiles.count; i++) {
            wait_tiles();
            if (i + 1 < tiles.count) fetch(i + 1);
            char* tile = smem + (i & 1) * 2 * H::kTileBytes;
            const int at = tiles[i] * H::kKeys;
            const Seen which = row0 < rows ? seen_of(a, wave_low, wave_high, at, H::kKeys) : kNone;
            if (!careful && which == kNone) continue;
#pragma unroll
            for (int b = 0; b < H::kKeyBlocks; b++) {
                u4 w[2];
                if (which != kNone) {
                    f16v s = f16v{}, dp = f16v{};
#pragma unroll
                    for (int k = 0; k < H::kSteps; k++) s = mfma32<DT>(read.rows(tile, b, k), q[k], s);
#pragma unroll
                    for (int k = 0; k < H::kSteps; k++) dp = mfma32<DT>(read.rows(tile + H::kTileBytes, b, k), grad[k], dp);
                    float ds[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) ds[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], a.scale, -lse)) * (dp[j] - delta);
                    if (which == kSome) {
#pragma unroll
                        for (int j = 0; j < 16; j++) ds[j] = sees(a, row.position, at + 32 * b + 8 * (j / 4) + 4 * half + j % 4) ? ds[j] : 0.f;
                    }
                    if constexpr (DT == BW_F16) fit_reach<16, H::kBlocks>(ds, reach, acc);
                    pack16<DT>(ds, w);
                }
                if (careful) {
                    __syncthreads();
                    if (which != kNone) add_nonfinite<H>(tile + b * 32 * H::kPitch * 2, 32, lane, acc, [&](int n) { return sees(a, row.position, at + 32 * b + n); });
                    keep_finite<H>(tile + b * 32 * H::kPitch * 2, 32 * H::kPitch * 2);
                }
                if (which != kNone) {
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int m = 0; m < H::kBlocks; m++) acc[m] = mfma32<DT>(read.columns(tile, 2 * b + t, m), w[t], acc[m]);
                }
            }
        }
        if (careful) break;
        float check = 0.f;
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
            for (int j = 0; j < 16; j++) check = __builtin_fmaf(acc[m][j], 0.f, check);
        if (!any_thread(smem, wave, row.live && check != 0.f)) break;
    }
    if (!row.live) return;
    const float back = DT == BW_F16 ? __builtin_ldexpf(1.f, -reach) : 1.f;
    uint16_t* out = g.q_grad + (token * a.q_heads + head * a.share + row.head) * a.dim;
#pragma unroll
    for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int d = 32 * m + 8 * b + 4 * half;
            const f4 x = f4{acc[m][4 * b], acc[m][4 * b + 1], acc[m][4 * b + 2], acc[m][4 * b + 3]} * back * g.plain_scale;
            if (d < a.dim) store4<DT>(out + d, x[0], x[1], x[2], x[3]);
        }
}

// A tile of rows of a sequence (tokens x the query heads of one key head) on its way to LDS; rows from the last on are the last one again.
template <class H> struct PackedLoader {
    uint32_t chunk[H::kLoads];
    int first;
    BW_DEV PackedLoader(int lane, int wave) {
        first = wave * H::kLoads * H::kLoadRows + lane / H::kChunks;
#pragma unroll
        for (int i = 0; i < H::kLoads; i++) chunk[i] = (uint32_t)((lane % H::kChunks) ^ swizzle<H::kPitch>(first + i * H::kLoadRows)) * 16;
    }
    BW_DEV void operator()(const PromptArgs& a, const uint16_t* base, int64_t row, int64_t head, int from, int rows, uint32_t to, int wave) const {
        to += wave * H::kLoads * 1024;
        uint32_t rest;
        const uint32_t token0 = a.by_share.div((uint32_t)from, rest);
        base += token0 * row;
        uint32_t bytes = (uint32_t)a.dim * 2;
        asm("" : "+s"(bytes));
#pragma unroll
        for (int i = 0; i < H::kLoads; i++) {
            const int r = from + first + i * H::kLoadRows;
            uint32_t j;
            const uint32_t token = a.by_share.div((uint32_t)(r < rows ? r : rows - 1), j);
            const uint32_t at = (token - token0) * (uint32_t)(2 * row) + j * (uint32_t)(2 * head) + chunk[i];
            if (chunk[i] < bytes) load_to_lds(base, at, to + i * 1024);
        }
    }
};
BW_DEV void load4_to_lds(const void* base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(base), "s"(to) : "memory");
}

// FAR: only rows that see the keys as sinks and not in their window, a share of them; otherwise only those that have them in their window (all, without a window).
template <class H, bool FAR>
__global__ __launch_bounds__(256, H::kResident) void prompt_key_grad_kernel(PromptGradArgs g) {
    extern __shared__ __align__(1024) char smem[];               // [2][Q, g, lse, delta]
    constexpr int DT = H::kType, kTileKeys = 32 * kPromptWaves, kStage = 2 * H::kTileBytes + 512, kTileRows = H::kKeys;
    const PromptArgs& a = g.p;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5;
    Span p;
    int head, sequence = 0;
    uint32_t split;
    if (FAR) {                                                   // a workgroup for a sequence, a tile of its sinks and a share of the rows
        uint32_t combo, s, h;
        uint32_t slot = a.by_combos.div(blockIdx.x, combo);
        split = slot % (uint32_t)g.far;
        slot /= (uint32_t)g.far;
        s = a.by_heads.div(combo, h);
        head = (int)h;
        sequence = (int)s;
        if (a.q_starts) {
            tokens_at(a.q_starts, sequence, a.sequences, a.q_tokens, p.q0, p.nq);
            tokens_at(a.k_starts, sequence, a.sequences, a.k_tokens, p.k0, p.nk);
            p.q0 = __builtin_amdgcn_readfirstlane(p.q0);
            p.nq = __builtin_amdgcn_readfirstlane(p.nq);
            p.k0 = __builtin_amdgcn_readfirstlane(p.k0);
            p.nk = __builtin_amdgcn_readfirstlane(p.nk);
        } else {
            p = Span{sequence * a.seq_q, a.seq_q, sequence * a.seq_k, a.seq_k, 0};
        }
        p.tile = (int)slot;
    } else {
        if (!place_of<kTileKeys, true>(a, p, head, split, &sequence)) return;
    }
    const int first = p.tile * kTileKeys, keys_all = FAR && a.sinks < p.nk ? a.sinks : p.nk, rows = p.nq * a.share, offset = p.nk - p.nq;
    if (FAR && first >= keys_all) return;
    clear_tiles<H>(smem, 2 * kStage, a.dim);
    const int key = first + wave * 32 + (lane & 31);
    const bool live = key < keys_all;
    const int64_t token = p.k0 + (live ? key : 0);
    u4 k[H::kSteps], v[H::kSteps];
    load_row<H>(k, a.k + token * a.k_row + head * a.k_head, live, a.dim, half);
    load_row<H>(v, a.v + token * a.v_row + head * a.v_head, live, a.dim, half);
#pragma unroll
    for (int s = 0; s < H::kSteps; s++)
#pragma unroll
        for (int j = 0; j < 4; j++) k[s][j] ^= a.flip;

    // Rows that count for a key: from ... to - 1 (positions key ... key + window - 1; further ones as a sink).
    auto row_at = [&](int64_t position) {
        const int64_t r = (position - offset) * a.share;
        return (int)(r < 0 ? 0 : r < rows ? r : rows);
    };
    auto rows_of = [&](int n, int& from, int& to) {
        from = row_at(FAR ? (int64_t)n + a.window : n);
        to = FAR ? rows : row_at((int64_t)n + a.window);
    };
    int row_from, row_to, from, to, other;
    rows_of(key, row_from, row_to);
    if (!live) row_from = row_to = 0;
    const int last = (first + kTileKeys < keys_all ? first + kTileKeys : keys_all) - 1;
    if (last < first) from = to = 0;
    else {
        rows_of(first, from, other);
        rows_of(last, other, to);
    }
    // ... for all of the wave's keys, and for any
    const int wave_first = first + wave * 32, wave_last = wave_first + 31 < last ? wave_first + 31 : last;
    int any_from = 0, any_to = 0, all_from = 0, all_to = 0;
    if (wave_first <= wave_last) {
        rows_of(wave_first, any_from, all_to);
        rows_of(wave_last, all_from, any_to);
    }
    const int tile_from = from / kTileRows, tile_count = to > from ? (to - 1) / kTileRows - tile_from + 1 : 0, pieces = FAR ? g.far : a.splits;
    const int begin = (int)((int64_t)tile_count * split / pieces), end = (int)((int64_t)tile_count * (split + 1) / pieces);

    const PackedLoader<H> load(lane, wave);
    const TileReader<H> read(lane);
    const uint16_t *queries = a.q + p.q0 * a.q_row + (int64_t)head * a.share * a.q_head, *grads = g.grad + p.q0 * g.grad_row + (int64_t)head * a.share * g.grad_head;
    const int64_t stats = (int64_t)head * a.q_tokens * a.share + (int64_t)p.q0 * a.share;
    const uint32_t lds = lds_address(smem);
    auto fetch = [&](int i) __attribute__((always_inline)) {
        const int at = (tile_from + i) * kTileRows;
        const uint32_t into = lds + (i & 1) * kStage;
        load(a, queries, a.q_row, a.q_head, at, rows, into, wave);
        load(a, grads, g.grad_row, g.grad_head, at, rows, into + H::kTileBytes, wave);
        const int r = at + lane < rows ? lane : rows - 1 - at;
        if (wave == 0) load4_to_lds(a.lse + stats + at, (uint32_t)r * 4, into + 2 * H::kTileBytes);
        if (wave == 1) load4_to_lds(g.delta + stats + at, (uint32_t)r * 4, into + 2 * H::kTileBytes + 256);
    };

    f16v dk[H::kBlocks], dv[H::kBlocks];
    int reach = 0;
    for (int careful = 0;; careful = 1) {
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++) dk[m] = dv[m] = f16v{};
        reach = kFirstReach16;
        if (begin < end) fetch(begin);
        for (int i = begin; i < end; i++) {
            wait_tiles();
            if (i + 1 < end) fetch(i + 1);
            char* tile = smem + (i & 1) * kStage;
            const int at = (tile_from + i) * kTileRows;
            const bool none = at >= any_to || at + kTileRows <= any_from, all = at >= all_from && at + kTileRows <= all_to;
            if (!careful && none) continue;
#pragma unroll
            for (int b = 0; b < kTileRows / 32; b++) {
                u4 pw[2], sw[2];
                if (!none) {
                    f16v s = f16v{}, dp = f16v{};
#pragma unroll
                    for (int n = 0; n < H::kSteps; n++) s = mfma32<DT>(read.rows(tile, b, n), k[n], s);
#pragma unroll
                    for (int n = 0; n < H::kSteps; n++) dp = mfma32<DT>(read.rows(tile + H::kTileBytes, b, n), v[n], dp);
                    float w[16], ds[16];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const f4 lse = *reinterpret_cast<const f4*>(tile + 2 * H::kTileBytes + (32 * b + 8 * j + 4 * half) * 4);
                        const f4 delta = *reinterpret_cast<const f4*>(tile + 2 * H::kTileBytes + 256 + (32 * b + 8 * j + 4 * half) * 4);
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            w[4 * j + n] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * j + n], a.scale, (DT == BW_F16 ? (float)kWeightShift : 0.f) - lse[n]));
                            ds[4 * j + n] = w[4 * j + n] * (dp[4 * j + n] - delta[n]);
                        }
                    }
                    if (!all) {
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const int r = at + 32 * b + 8 * (j / 4) + 4 * half + j % 4;
                            const bool counts = r >= row_from && r < row_to;
                            w[j] = counts ? w[j] : 0.f;
                            ds[j] = counts ? ds[j] : 0.f;
                        }
                    }
                    if constexpr (DT == BW_F16) fit_reach<16, H::kBlocks>(ds, reach, dk);
                    pack16<DT>(w, pw);
                    pack16<DT>(ds, sw);
                }
                if (careful) {
                    char *qs = tile + b * 32 * H::kPitch * 2, *gs = qs + H::kTileBytes;
                    __syncthreads();
                    if (!none) {
                        auto counts = [&](int n) { return at + 32 * b + n >= row_from && at + 32 * b + n < row_to; };
                        add_nonfinite<H>(qs, 32, lane, dk, counts);
                        add_nonfinite<H>(gs, 32, lane, dv, counts);
                    }
                    keep_finite<H>(qs, 32 * H::kPitch * 2);
                    keep_finite<H>(gs, 32 * H::kPitch * 2);
                }
                if (!none) {
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int m = 0; m < H::kBlocks; m++) dv[m] = mfma32<DT>(read.columns(tile + H::kTileBytes, 2 * b + t, m), pw[t], dv[m]);
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int m = 0; m < H::kBlocks; m++) dk[m] = mfma32<DT>(read.columns(tile, 2 * b + t, m), sw[t], dk[m]);
                }
            }
        }
        if (careful) break;
        float check = 0.f;
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
            for (int j = 0; j < 16; j++) check = __builtin_fmaf(dv[m][j], 0.f, __builtin_fmaf(dk[m][j], 0.f, check));
        if (!any_thread(smem, wave, live && check != 0.f)) break;
    }
    if (!live) return;
    const float k_by = g.plain_scale * (DT == BW_F16 ? __builtin_ldexpf(1.f, -reach - kWeightShift) : 1.f), v_by = DT == BW_F16 ? __builtin_ldexpf(1.f, -kWeightShift) : 1.f;
    const int64_t sink_at = ((int64_t)(sequence * a.kv_heads + head) * g.far * a.sinks + key) * 2 * a.dim;
    float* part = FAR ? g.sink_parts + sink_at + (int64_t)split * a.sinks * 2 * a.dim
                      : a.splits > 1 ? g.parts + (((int64_t)split * a.k_tokens + token) * a.kv_heads + head) * 2 * a.dim : nullptr;
    const bool sinks = !FAR && g.far && split == 0 && key < a.sinks && sequence < a.sequences;
#pragma unroll
    for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int d = 32 * m + 8 * b + 4 * half;
            if (d >= a.dim) continue;
            f4 x = f4{dk[m][4 * b], dk[m][4 * b + 1], dk[m][4 * b + 2], dk[m][4 * b + 3]} * k_by, y = f4{dv[m][4 * b], dv[m][4 * b + 1], dv[m][4 * b + 2], dv[m][4 * b + 3]} * v_by;
            if (sinks) {
                for (int n = 0; n < g.far; n++) {
                    const float* from = g.sink_parts + sink_at + (int64_t)n * a.sinks * 2 * a.dim + d;
                    x += *reinterpret_cast<const f4*>(from);
                    y += *reinterpret_cast<const f4*>(from + a.dim);
                }
            }
            if (part) {
                *reinterpret_cast<f4*>(part + d) = x;
                *reinterpret_cast<f4*>(part + a.dim + d) = y;
            } else {
                const int64_t to_at = (token * a.kv_heads + head) * a.dim + d;
                if (g.k_grad) store4<DT>(g.k_grad + to_at, x[0], x[1], x[2], x[3]);
                if (g.v_grad) store4<DT>(g.v_grad + to_at, y[0], y[1], y[2], y[3]);
            }
        }
}
