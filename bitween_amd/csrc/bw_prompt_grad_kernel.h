// bw_prompt_grad_kernel.h - gradients of the attention in bw_prompt_kernel.h.  With P = 2^(S c - lse), the weights of the forward again, and g the output's gradient:
//   dP = g V^T,  delta = rowsum(g out),  dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T g
// One kernel has the rows and goes over the keys (dQ, and delta on the way), another has the keys and goes over the rows (dK, dV), so that every sum is a
// workgroup's own, in one order: eight products where five would do with sums in memory, and the same bits every time.
//
// P and dS enter their second product as 16-bit numbers, rounded once (as in the forward, at the same price of a second product for each).  lse is that of the forward's rounded weights, so that a
// row's P add up to 1 but for half a step at most (of a few keys; where there are many the roundings cancel); a float32 sum beside it would cost the forward 5 % (heads of 64 9 %), one here some 15
// registers, which go to memory.  In float16, whose steps end at 2^-24, P goes in 2^12 times as large, and dS times a power of two that
// is each row's (each key's) own: it starts high and comes down where a product would pass 2^15, and the sums with it.
//
// A row's dS add up to zero, but for what dS and the output (in delta) were rounded by: a remainder e, which puts e times the mean of the keys into dQ.  Keys are projected with
// channels far from zero, so that this was the larger part of dQ's error (8192 tokens, bfloat16, channels at 2 to 6 of keys that spread by 1: 0.0045 of dQ, 0.0024 without it; 2 tokens: 0.0060 and 0.0025).
// dQ = scale dS (K - c) for any c: e is summed as the product takes it, and e c taken off, c the mean of the last 32 keys that a row sees.
// What the dS add up to before they are rounded is what the rounded output is off by in delta (the weights of a row add up to 1): the rows' kernel, which sees all keys, hands delta on to dK
// without it (dK's error, 2 tokens: 0.0039 with it, 0.0024 without); where keys are in parts each leaves its sum, and the join takes them off.
//
// What bounds them is what bounds the forward; matrix cores busy 49 ... 51 % (dQ) and 46 % (dK, dV), vector unit 42 and 36 %.  8192 tokens, 32 and 8 heads of 128, bfloat16: dQ 770 ... 840 us (1075 ... 980 TFLOP/s
// of its three products, as the clocks of cards differ), dK and dV 1300 ... 1420 (1060 ... 970 of their five), 2075 ... 2260 in all.
#pragma once
#include "bw_prompt_kernel.h"

struct PromptGradArgs {
    PromptArgs p;
    const uint16_t *grad, *result;               // of the output; result [tokens][q_heads][dim]
    int64_t grad_row, grad_head;
    float* delta;                                // its negative, as lse
    int exact;                                   // delta is wanted that is that of the weights, not of the rounded result (see above)
    uint16_t *q_grad, *k_grad, *v_grad;
    float *q_parts, *q_left;                     // where a row's keys are cut into p.splits parts: [row][part][dim], and sums of their dS [row][part]
    float plain_scale;
    // keys: the list of the workgroups' pieces (NULL: a piece for every tile of keys), the parts [part][kv_heads][keys][2][dim] and what is to be joined of them
    struct KeyPlan* plan;
    struct Piece* pieces;
    struct KeyJoin* joins;
    int* tiles_before;                           // of sequence s: where its tiles of keys begin
    float* parts;
    int target;                                  // pieces (of one head) that the rows are cut into, about
    int room, parts_room, joins_room;            // of the lists
    uint32_t before;                             // workgroups in the launches before this one (see in_launches)
};

constexpr int kFirstReach16 = 80, kReachTop = 12, kReachMost = 15, kWeightShift = 12;

// The power of two (of each lane) that its values `x`, times 2^reach, go into a product with, which brings down the sums in `acc` where it comes down.
template <int N, int BLOCKS> BW_DEV void fit_reach(float* x, int& reach, f16v* acc, float& sum) {
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
        sum *= by;
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

// ---- the list of pieces of the keys' gradients (see key_grad) ----

// A piece has at least so many tiles of rows.
constexpr int kLeastTiles = 4;


constexpr int kGradKeys = 32 * kPromptWaves;

// Tiles from ... to - 1 of rows (kKeys each) for the keys from kGradKeys tile on of a sequence; part: which of the parts they leave, or -1.
struct Piece { int q0, nq, k0, nk, tile, from, to, part; };
// Keys whose parts are to be added up.
struct KeyJoin { int key, keys, part, parts; };
struct KeyPlan { int pieces, joins; };

// Rows of a sequence that see a key: from ... to - 1.
BW_DEV void rows_of_key(const PromptArgs& a, int nq, int nk, int key, int& from, int& to) {
    auto row_at = [&](int64_t position) {
        const int64_t r = (position - (nk - nq)) * a.share, rows = (int64_t)nq * a.share;
        return (int)(r < 0 ? 0 : r < rows ? r : rows);
    };
    from = row_at(key);
    to = key < a.sinks ? nq * a.share : row_at((int64_t)key + a.window);
}
// Tiles of rows that a tile of keys meets.
BW_DEV void tiles_of_keys(const PromptArgs& a, int nq, int nk, int tile, int tile_rows, int& from, int& to) {
    const int first = tile * kGradKeys, last = (first + kGradKeys < nk ? first + kGradKeys : nk) - 1;
    int begin, end, other;
    rows_of_key(a, nq, nk, first, begin, end);
    rows_of_key(a, nq, nk, last, other, other);
    end = end > other ? end : other;
    from = begin / tile_rows;
    to = end > begin ? (end - 1) / tile_rows + 1 : from;
}

constexpr int kPlanThreads = 256;
// Sum of the threads' numbers before this one's, and of all.
BW_DEV int sum_before(int* lds, int mine, int& all) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int other = __shfl_up(sum, o, 64);
        if (lane >= o) sum += other;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    int before = sum - mine;
    all = 0;
    for (int w = 0; w < kPlanThreads / 64; w++) {
        if (w < wave) before += lds[w];
        all += lds[w];
    }
    return before;
}

// Every tile of keys in pieces of at most so many tiles of rows that there are about g.target pieces; by one workgroup.
BW_DEV void plan_keys(const PromptGradArgs& g, char* smem, int tile_rows) {
    int* lds = reinterpret_cast<int*>(smem);
    unsigned long long& units = *reinterpret_cast<unsigned long long*>(smem + 64);
    const int least = kLeastTiles;
    const PromptArgs& a = g.p;
    const int sequences = a.q_starts ? a.sequences + 2 : a.sequences, thread = (int)threadIdx.x;
    auto tokens = [&](int s, Piece& p) {
        if (a.q_starts) {
            tokens_at(a.q_starts, s, a.sequences, a.q_tokens, p.q0, p.nq);
            tokens_at(a.k_starts, s, a.sequences, a.k_tokens, p.k0, p.nk);
            if (s >= a.sequences) p.nq = 0;
        } else {
            p.q0 = s * a.seq_q; p.nq = a.seq_q; p.k0 = s * a.seq_k; p.nk = a.seq_k;
        }
    };
    int& decreases = *reinterpret_cast<int*>(smem + 72);
    if (thread == 0) {
        units = 0;
        decreases = 0;
    }
    __syncthreads();
    int tiles = 0;
    for (int base = 0; base < sequences; base += kPlanThreads) {
        const int s = base + thread;
        Piece p = {};
        if (s < sequences) tokens(s, p);
        if (a.q_starts && s < a.sequences && start_at(a.k_starts, s + 1, a.k_tokens) < start_at(a.k_starts, s, a.k_tokens)) decreases = 1;
        int all;
        const int before = tiles + sum_before(lds, (p.nk + kGradKeys - 1) / kGradKeys, all);
        if (s < sequences) g.tiles_before[s] = before;
        tiles += all;
    }
    __syncthreads();                                             // (and its fence: tiles_before is read below)
    if (decreases) tiles = 0;                                    // (the same tokens over and over, more than can be counted: no gradients then)
    auto piece_of = [&](int n) {                                 // the n-th tile of keys
        int lo = 0, hi = sequences;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (g.tiles_before[mid] <= n) lo = mid;
            else hi = mid;
        }
        Piece p = {};
        tokens(lo, p);
        p.tile = n - g.tiles_before[lo];
        tiles_of_keys(a, p.nq, p.nk, p.tile, tile_rows, p.from, p.to);
        return p;
    };
    unsigned long long mine = 0;
    for (int n = thread; n < tiles; n += kPlanThreads) {
        const Piece p = piece_of(n);
        mine += (unsigned)(p.to - p.from);
    }
    atomicAdd(&units, mine);                                     // (whole numbers: any order gives the same)
    __syncthreads();
    const unsigned long long each = (units + g.target - 1) / g.target;
    const int size = each > (unsigned)least ? (int)each : least;
    int pieces = 0, parts = 0, joins = 0;
    for (int base = 0; base < tiles; base += kPlanThreads) {
        const int n = base + thread;
        Piece p = {};
        int cuts = 0;
        if (n < tiles) {
            p = piece_of(n);
            const int tiles_of_rows = p.to - p.from;
            cuts = (tiles_of_rows - tiles_of_rows / 4 + size - 1) / size;        // (a third longer rather than cut: parts cost a way through memory)
            if (cuts < 1) cuts = 1;
        }
        int all_pieces, all_parts, all_joins;
        const int piece = pieces + sum_before(lds, cuts, all_pieces), part = parts + sum_before(lds, cuts > 1 ? cuts : 0, all_parts), join = joins + sum_before(lds, cuts > 1, all_joins);
        const bool whole = cuts > 1 && (part + cuts > g.parts_room || join >= g.joins_room);
        for (int c = 0; c < cuts && piece + c < g.room; c++) {
            Piece one = p;
            if (!whole) {
                one.from = p.from + (int)((int64_t)(p.to - p.from) * c / cuts);
                one.to = p.from + (int)((int64_t)(p.to - p.from) * (c + 1) / cuts);
            } else if (c) {
                one.nk = 0;                                      // nothing
                one.to = one.from;
            }
            one.part = cuts > 1 && !whole ? part + c : -1;
            g.pieces[piece + c] = one;
        }
        if (cuts > 1 && join < g.joins_room) g.joins[join] = whole ? KeyJoin{0, 0, 0, 0} : KeyJoin{p.k0 + p.tile * kGradKeys, p.nk - p.tile * kGradKeys < kGradKeys ? p.nk - p.tile * kGradKeys : kGradKeys, part, cuts};
        pieces += all_pieces;
        parts += all_parts;
        joins += all_joins;
    }
    if (thread == 0) *g.plan = KeyPlan{pieces < g.room ? pieces : g.room, joins < g.joins_room ? joins : g.joins_room};
}

// Beside the queries' gradient, whose workgroups it is hidden among, the first workgroup lists the pieces of the keys' (on its own, in between: 14 us).
template <class H>
__global__ __launch_bounds__(256, H::kPitch == 64 ? 3 : H::kResident) void prompt_query_grad_kernel(PromptGradArgs g) {
    extern __shared__ __align__(1024) char smem[];               // [2][K, V]
    constexpr int DT = H::kType;
    const PromptArgs& a = g.p;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5;
    Span p;
    int head;
    uint32_t split;
    const uint32_t block = g.before + blockIdx.x;
    if (g.plan && block == 0) {
        plan_keys(g, smem, H::kKeys);
        return;
    }
    if (!place_of<kRows, false>(a, g.plan ? block - 1 : block, p, head, split)) return;
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
    if ((!g.exact || a.splits > 1) && row.live && half == 0 && split == 0) g.delta[index] = -delta;
    if (!g.exact) return;
    const float lse = row.live ? a.lse[index] : INFINITY;

    int low, high, wave_low, wave_high;
    positions_of(a, p, p.tile * kRows, (p.tile + 1) * kRows, low, high);
    positions_of(a, p, row0 < rows ? row0 : p.tile * kRows, row0 + kWaveRows, wave_low, wave_high);
    const KeyTiles tiles(a, low, high, p.nk, H::kKeys);
    int begin, end;
    tiles.part(a, split, begin, end);
    const RowLoader<H> load_k(a, lane, wave, a.k_row), load_v(a, lane, wave, a.v_row);
    const TileReader<H> read(lane);
    const SeenOf<H::kKeys> seen(a, wave_low, wave_high, row0 < rows);
    const uint32_t lds = own(lds_address(smem));
    const int keys = own(p.nk);
    const float scale = own(a.scale);
    auto fetch = [&](const KeyWalk<H>& next) __attribute__((always_inline)) {
        const uint32_t to = lds + (next.i & 1) * 2 * H::kTileBytes;
        load_k(next.k, keys - next.at, to, wave);
        load_v(next.v, keys - next.at, to + H::kTileBytes, wave);
    };

    f16v acc[H::kBlocks];
    int reach = 0;
    float rest = 0.f, left = 0.f;                                // sums of the dS, as rounded and before
    auto pass = [&](auto is_careful) __attribute__((always_inline)) {       // (see prompt_forward_kernel)
        constexpr bool careful = decltype(is_careful)::value;
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++) acc[m] = f16v{};
        reach = kFirstReach16;
        rest = left = 0.f;
        KeyWalk<H> next(a, p, head, tiles, begin);
        if (begin < end) fetch(next);
        for (int i = begin; i < end; i++) {
            const int at = next.at;
            next.step();
            wait_tiles();
            if (next.i < end) fetch(next);
            char* tile = smem + (i & 1) * 2 * H::kTileBytes;
            const int which = seen(at);
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
                    reads_ahead<2 * H::kSteps, 1, 4>();
                    float ds[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) ds[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], scale, -lse)) * (dp[j] - delta);
                    if (which != kAll) hide<16>(which, a, row.position, at + 32 * b + 4 * half, 0.f, ds);
#pragma unroll
                    for (int j = 0; j < 16; j++) left += ds[j];
                    if constexpr (DT == BW_F16) fit_reach<16, H::kBlocks>(ds, reach, acc, rest);
                    pack16<DT>(ds, w);
#pragma unroll
                    for (int j = 0; j < 8; j++) rest = add_pair<DT>(w[j / 4][j % 4], rest);
                }
                if constexpr (careful) {
                    __syncthreads();
                    if (which != kNone) add_nonfinite<H>(tile + b * 32 * H::kPitch * 2, 32, lane, acc, [&](int n) { return sees(a, row.position, at + 32 * b + n); });
                    keep_finite<H>(tile + b * 32 * H::kPitch * 2, 32 * H::kPitch * 2);
                }
                if (which != kNone) {                            // (with the first of these operands read before the weights, as for the keys below: no gain with heads of 128, a tenth lost with 64 and 256)
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int m = 0; m < H::kBlocks; m++) acc[m] = mfma32<DT>(read.columns(tile, 2 * b + t, m), w[t], acc[m]);
                }
            }
        }
    };
    pass(std::false_type{});
    const bool some = any_thread(smem, wave, row.live && not_finite<H::kBlocks>(acc));
    if (some) pass(std::true_type{});
    rest += __shfl_xor(rest, 32, 64);
    left += __shfl_xor(left, 32, 64);
    if (row.live && half == 0) {
        if (a.splits > 1) g.q_left[index * a.splits + split] = left;
        else g.delta[index] = -(delta + left);
    }
    if (!g.q_grad) return;
    const float back = DT == BW_F16 ? __builtin_ldexpf(1.f, -reach) : 1.f;
    uint16_t* out = g.q_grad + (token * a.q_heads + head * a.share + row.head) * a.dim;
    float* part = a.splits > 1 ? g.q_parts + (index * a.splits + split) * a.dim : nullptr;
    // c: of each row the mean of the last 32 keys at most that it sees, by a product with weights of 1 / n (rounded to the type: any c will do); of the up to 63 keys of a wave's rows in two
    // steps.  Infinities and NaN are left out, where there may be any: each of these keys is seen by a row of the wave, and where one workgroup goes over all keys a row that sees one has
    // no finite sum.  Where they are cut into parts the key lies in another's, which puts it into that row's dQ; here it would reach the rows before it.
    const bool finite_only = some || a.splits > 1;
    __syncthreads();
    char* mine = smem + wave * 32 * H::kPitch * 2;
    const int last = row.position, windowed = last - a.window + 1, from = windowed > last - 31 ? windowed > 0 ? windowed : 0 : last > 31 ? last - 31 : 0;
    const int lowest = wave_low - (a.window < 32 ? a.window : 32) + 1, first_key = lowest > 0 ? lowest : 0, chunk = lane % H::kChunks;
    const float one = last >= from ? 1.f / (float)(last - from + 1) : 0.f;
    constexpr int kAtOnce = H::kBlocks < 4 ? H::kBlocks : 4;
#pragma unroll
    for (int m0 = 0; m0 < H::kBlocks; m0 += kAtOnce) {
        f16v mean[kAtOnce];
#pragma unroll
        for (int m = 0; m < kAtOnce; m++) mean[m] = f16v{};
#pragma unroll 1
        for (int base = first_key; base <= first_key + 32; base += 32) {
#pragma unroll
            for (int i = 0; i < 32 / H::kLoadRows; i++) {
                const int n = i * H::kLoadRows + lane / H::kChunks;
                u4 v = {0, 0, 0, 0};
                if (base + n <= wave_high && chunk * 8 < a.dim) v = *reinterpret_cast<const u4*>(a.k + (int64_t)(p.k0 + base + n) * a.k_row + head * a.k_head + chunk * 8);
                if (finite_only) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t w = v[j];
                        v[j] = (finite16<DT>(w) ? w & 0xFFFFu : 0u) | (finite16<DT>(w >> 16) ? w & 0xFFFF0000u : 0u);
                    }
                }
                *reinterpret_cast<u4*>(mine + n * H::kPitch * 2 + (chunk ^ swizzle<H::kPitch>(n)) * 16) = v;
            }
            __syncthreads();
            float x[16];
            u4 w[2];
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int key = base + 8 * (j / 4) + 4 * half + j % 4;
                x[j] = key >= from && key <= last ? one : 0.f;
            }
            pack16<DT>(x, w);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int m = 0; m < kAtOnce; m++) mean[m] = mfma32<DT>(read.columns(mine, t, m0 + m), w[t], mean[m]);
            __syncthreads();
        }
        if (row.live) {
#pragma unroll
            for (int m = 0; m < kAtOnce; m++)
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const int d = 32 * (m0 + m) + 8 * b + 4 * half;
                    f4 x;
#pragma unroll
                    for (int i = 0; i < 4; i++) x[i] = (acc[m0 + m][4 * b + i] - rest * mean[m][4 * b + i]) * back * g.plain_scale;
                    if (d >= a.dim) continue;
                    if (part) *reinterpret_cast<f4*>(part + d) = x;
                    else store4<DT>(out + d, x[0], x[1], x[2], x[3]);
                }
        }
    }
}

// dQ = the parts of a row added up in order, and delta without what their dS add up to; a thread has 4 values of a row, and 8 parts under way.
template <int DT>
__global__ __launch_bounds__(256) void prompt_query_join_kernel(PromptGradArgs g, int threads, uint32_t rows) {
    const PromptArgs& a = g.p;
    const uint32_t i = blockIdx.x * (256 / threads) + threadIdx.x / threads;
    const int d = (int)(threadIdx.x % threads) * 4;
    if (threadIdx.x / threads >= 256 / threads || i >= rows) return;
    const float *part = g.q_parts + (int64_t)i * a.splits * a.dim + d, *lefts = g.q_left + (int64_t)i * a.splits;
    f4 o = {0.f, 0.f, 0.f, 0.f};
    float left = 0.f;
    for (int s = 0; s < a.splits; s += 8) {
        f4 x[8];
        float y[8];
#pragma unroll
        for (int n = 0; n < 8; n++) {
            const int at = s + n < a.splits ? s + n : s;
            y[n] = lefts[at];
            if (g.q_grad) x[n] = *reinterpret_cast<const f4*>(part + (int64_t)at * a.dim);
        }
#pragma unroll
        for (int n = 0; n < 8; n++) {
            if (s + n >= a.splits) continue;
            left += y[n];
            if (g.q_grad) o += x[n];
        }
    }
    if (d == 0) g.delta[i] -= left;
    if (!g.q_grad) return;
    uint32_t j;
    const uint32_t token_head = a.by_share.div(i, j), head = token_head / (uint32_t)a.q_tokens, token = token_head - head * a.q_tokens;
    store4<DT>(g.q_grad + ((int64_t)token * a.q_heads + head * a.share + j) * a.dim + d, o[0], o[1], o[2], o[3]);
}

// ---- keys ----
//
// A workgroup has 128 keys of one sequence and one key head, 32 to a wave, and the rows come by, kKeys at a time: S and dP with a key to a lane, so that P and dS are the
// second operands of dV^T += g^T P and dK^T += Q^T dS as they lie.  dV and dK are workgroups of their own, side by side in one launch, though both need S: one wave with
// both sums does not fit two workgroups to a CU (of 256 registers, 64 of operands and 128 of sums leave too few: 283 TFLOP/s with 250 bytes of a lane in memory; one workgroup, with 512, has not been
// tried), and two waves that share S and P through LDS
// wait for each other every 32 rows (8192 tokens, 32 and 8 heads of 128: 2068 us).
//
// Rows are cut into pieces of equal length, each a workgroup's: a workgroup lists them first (plan_keys), since a key that is seen by all rows meets many times the
// rows of the last one.  The parts of keys that several workgroups have are added up in order by prompt_grad_join_kernel.
// Tiles of rows of a sequence (tokens x the query heads of one key head) on their way to LDS; rows from the last on are the last one again.  Where a tile is
// whole tokens, as it is for 1, 2, 4 ... query heads to a key head, a lane's place in it stays the same.
template <class H> struct PackedLoader {
    uint32_t place[H::kLoads], chunk[H::kLoads];
    int first, same_to;                          // row of the lane in the first load; tiles that begin before it are whole ones of such tokens
    uint32_t step, row_bytes, head_bytes, bytes;
    const char* base;
    BW_DEV PackedLoader(const PromptArgs& a, int lane, int wave, const uint16_t* from, int64_t row, int64_t head, int rows) {
        first = wave * H::kLoads * H::kLoadRows + lane / H::kChunks;
        uint32_t j;
        const int tokens = (int)a.by_share.div((uint32_t)H::kKeys, j);
        same_to = own(j == 0 ? rows - H::kKeys + 1 : 0);
        step = own((uint32_t)(2 * tokens * row));                // (rows are 2^24 - 1 apart at most, and a key head's query heads 2^31)
        row_bytes = own((uint32_t)(2 * row));
        head_bytes = own((uint32_t)(2 * head));
        bytes = own((uint32_t)a.dim * 2);
        base = own((const char*)from);
#pragma unroll
        for (int i = 0; i < H::kLoads; i++) {
            const int r = first + i * H::kLoadRows;
            chunk[i] = (uint32_t)((lane % H::kChunks) ^ swizzle<H::kPitch>(r)) * 16;
            const uint32_t token = a.by_share.div((uint32_t)r, j);
            place[i] = token * row_bytes + j * head_bytes + chunk[i];
        }
    }
    BW_DEV void operator()(const PromptArgs& a, int tile, int rows, uint32_t to, int wave) const {
        const int from = tile * H::kKeys;
        to += wave * H::kLoads * 1024;
        uint32_t some = bytes;
        asm("" : "+s"(some));                                    // (the comparisons below are not kept in registers over the loop)
        if (from < same_to) {
            const char* here = base + (uint64_t)step * (uint32_t)tile;
            if (some == H::kPitch * 2) {
#pragma unroll
                for (int i = 0; i < H::kLoads; i++) load_to_lds(here, place[i], to + i * 1024);
            } else {
#pragma unroll
                for (int i = 0; i < H::kLoads; i++)
                    if (chunk[i] < some) load_to_lds(here, place[i], to + i * 1024);
            }
            return;
        }
        uint32_t rest;
        const uint32_t token0 = a.by_share.div((uint32_t)from, rest);
        const char* here = base + (uint64_t)row_bytes * token0;
#pragma unroll
        for (int i = 0; i < H::kLoads; i++) {
            const int r = from + first + i * H::kLoadRows;
            uint32_t j;
            const uint32_t token = a.by_share.div((uint32_t)(r < rows ? r : rows - 1), j);
            if (chunk[i] < some) load_to_lds(here, (token - token0) * row_bytes + j * head_bytes + chunk[i], to + i * 1024);
        }
    }
};

// sums += the transposed product of 32 rows of a tile with the 16 + 16 values of a lane: the second 16's operands are read while the first products are under way.  `first`: the first
// 16's, read by then.
template <class H> BW_DEV void first_columns(const TileReader<H>& read, const char* tile, int block, u4* first) {
#pragma unroll
    for (int m = 0; m < H::kBlocks; m++) first[m] = read.columns(tile, 2 * block, m);
}
template <class H> BW_DEV void add_columns(const TileReader<H>& read, const char* tile, int block, const u4* first, const u4* w, f16v* acc) {
    in_order();
    u4 second[H::kBlocks];
#pragma unroll
    for (int m = 0; m < H::kBlocks; m++) second[m] = read.columns(tile, 2 * block + 1, m);
#pragma unroll
    for (int m = 0; m < H::kBlocks; m++) acc[m] = mfma32<H::kType>(first[m], w[0], acc[m]);
    in_order();
#pragma unroll
    for (int m = 0; m < H::kBlocks; m++) acc[m] = mfma32<H::kType>(second[m], w[1], acc[m]);
}

template <class H> constexpr int kKeyStage = 2 * H::kTileBytes + 512;           // Q, g, lse, delta of a tile of rows

// One piece: dK of its keys, or dV.
template <class H, bool DK> BW_DEV void key_grad(const PromptGradArgs& g, const Piece& p, int head, char* smem) {
    constexpr int DT = H::kType, kTileRows = H::kKeys;
    const PromptArgs& a = g.p;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5;
    const int rows = p.nq * a.share, wave_first = p.tile * kGradKeys + wave * 32, key = wave_first + (lane & 31);
    const bool live = key < p.nk;
    const int64_t token = p.k0 + (live ? key : 0);
    u4 k[H::kSteps], v[DK ? H::kSteps : 1];
    load_row<H>(k, a.k + token * a.k_row + head * a.k_head, live, a.dim, half);
    if constexpr (DK) load_row<H>(v, a.v + token * a.v_row + head * a.v_head, live, a.dim, half);
#pragma unroll
    for (int s = 0; s < H::kSteps; s++)
#pragma unroll
        for (int j = 0; j < 4; j++) k[s][j] ^= a.flip;

    // Rows that count for the lane's key; for any of the wave's; for all of them.
    int row_from = 0, row_to = 0, any_from = 0, any_to = 0, all_from = 0, all_to = 0;
    if (live) rows_of_key(a, p.nq, p.nk, key, row_from, row_to);
    if (wave_first < p.nk) {
        const int wave_last = wave_first + 31 < p.nk ? wave_first + 31 : p.nk - 1;
        int first_to, last_to, ignored;
        rows_of_key(a, p.nq, p.nk, wave_first, any_from, first_to);
        rows_of_key(a, p.nq, p.nk, wave_last, all_from, last_to);
        any_to = first_to > last_to ? first_to : last_to;
        // (the first key that is no sink leaves its window first)
        rows_of_key(a, p.nq, p.nk, a.sinks > wave_first && a.sinks <= wave_last ? a.sinks : wave_first, ignored, all_to);
    }

    const TileReader<H> read(lane);
    const uint16_t *queries = a.q + p.q0 * a.q_row + (int64_t)head * a.share * a.q_head, *grads = g.grad + p.q0 * g.grad_row + (int64_t)head * a.share * g.grad_head;
    any_from = own(any_from);
    any_to = own(any_to);
    all_from = own(all_from);
    all_to = own(all_to);
    const float scale = own(a.scale);
    const int begin = own(p.from), end = own(p.to);
    const int64_t stats = (int64_t)head * a.q_tokens * a.share + (int64_t)p.q0 * a.share;
    const uint32_t lds = lds_address(smem);
    const PackedLoader<H> load_q(a, lane, wave, queries, a.q_row, a.q_head, rows), load_g(a, lane, wave, grads, g.grad_row, g.grad_head, rows);
    auto fetch = [&](int i) __attribute__((always_inline)) {
        const int at = i * kTileRows;
        const uint32_t into = lds + (i & 1) * kKeyStage<H>;
        load_q(a, i, rows, into, wave);
        load_g(a, i, rows, into + H::kTileBytes, wave);
        const int r = at + lane < rows ? lane : rows - 1 - at;
        if (wave == 0) load4_to_lds(a.lse + stats + at, (uint32_t)r * 4, into + 2 * H::kTileBytes);
        if (DK && wave == 1) load4_to_lds(g.delta + stats + at, (uint32_t)r * 4, into + 2 * H::kTileBytes + 256);
    };

    f16v acc[H::kBlocks];
    int reach = 0;
    auto pass = [&](auto is_careful) __attribute__((always_inline)) {       // (see prompt_forward_kernel)
        constexpr bool careful = decltype(is_careful)::value;
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++) acc[m] = f16v{};
        reach = kFirstReach16;
        if (begin < end) fetch(begin);
        for (int i = begin; i < end; i++) {
            wait_tiles();
            if (i + 1 < end) fetch(i + 1);
            char* tile = smem + (i & 1) * kKeyStage<H>;
            const int at = i * kTileRows;
            const bool none = at >= any_to || at + kTileRows <= any_from, all = at >= all_from && at + kTileRows <= all_to;
            if (!careful && none) continue;
#pragma unroll
            for (int b = 0; b < kTileRows / 32; b++) {
                u4 w[2], first[H::kBlocks];
                char* from = tile + (DK ? 0 : H::kTileBytes);
                if (!none) {
                    const char* stat = tile + 2 * H::kTileBytes + (32 * b + 4 * half) * 4;
                    f16v s = f16v{}, dp = f16v{};
                    in_order();
                    if constexpr (DK) {                            // dP - delta: the sums begin at -delta
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const f4 delta = *reinterpret_cast<const f4*>(stat + 256 + 32 * j);
#pragma unroll
                            for (int n = 0; n < 4; n++) dp[4 * j + n] = delta[n];
                        }
                        in_order();
                    }
#pragma unroll
                    for (int n = 0; n < H::kSteps; n++) s = mfma32<DT>(read.rows(tile, b, n), k[n], s);
                    if constexpr (DK) {
#pragma unroll
                        for (int n = 0; n < H::kSteps; n++) dp = mfma32<DT>(read.rows(tile + H::kTileBytes, b, n), v[n], dp);
                    }
                    reads_ahead<(DK ? 2 : 1) * H::kSteps, 1, 4>();
                    in_order();
                    f4 lses[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) lses[j] = *reinterpret_cast<const f4*>(stat + 32 * j);
                    if constexpr (!careful) first_columns<H>(read, from, b, first);
                    float x[16];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * j + n], scale, (DT == BW_F16 ? (float)kWeightShift : 0.f) - lses[j][n]));
                            x[4 * j + n] = DK ? p * dp[4 * j + n] : p;
                        }
                    }
                    if (!all) {
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const int r = at + 32 * b + 8 * (j / 4) + 4 * half + j % 4;
                            x[j] = r >= row_from && r < row_to ? x[j] : 0.f;
                        }
                    }
                    if constexpr (DK && DT == BW_F16) {
                        float none = 0.f;
                        fit_reach<16, H::kBlocks>(x, reach, acc, none);
                    }
                    pack16<DT>(x, w);
                }
                if constexpr (careful) {
                    char* block = from + b * 32 * H::kPitch * 2;
                    __syncthreads();
                    if (!none) add_nonfinite<H>(block, 32, lane, acc, [&](int n) { return at + 32 * b + n >= row_from && at + 32 * b + n < row_to; });
                    keep_finite<H>(block, 32 * H::kPitch * 2);
                    if (!none) first_columns<H>(read, from, b, first);
                }
                if (!none) add_columns<H>(read, from, b, first, w, acc);
            }
        }
    };
    pass(std::false_type{});
    if (any_thread(smem, wave, live && not_finite<H::kBlocks>(acc))) pass(std::true_type{});
    if (!live) return;
    const float by = (DK ? g.plain_scale : 1.f) * (DT == BW_F16 ? __builtin_ldexpf(1.f, -kWeightShift - (DK ? reach : 0)) : 1.f);
    float* part = p.part < 0 ? nullptr : g.parts + ((((int64_t)p.part * a.kv_heads + head) * kGradKeys + key - p.tile * kGradKeys) * 2 + DK) * a.dim;
    uint16_t* out = (DK ? g.k_grad : g.v_grad) + (token * a.kv_heads + head) * a.dim;
#pragma unroll
    for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int d = 32 * m + 8 * b + 4 * half;
            const f4 x = f4{acc[m][4 * b], acc[m][4 * b + 1], acc[m][4 * b + 2], acc[m][4 * b + 3]} * by;
            if (d >= a.dim) continue;
            if (part) *reinterpret_cast<f4*>(part + d) = x;
            else store4<DT>(out + d, x[0], x[1], x[2], x[3]);
        }
}

template <class H>
__global__ __launch_bounds__(256, H::kResident) void prompt_key_grad_kernel(PromptGradArgs g) {
    extern __shared__ __align__(1024) char smem[];               // [2][Q, g, lse, delta]
    const PromptArgs& a = g.p;
    // Neighbouring workgroups, which go to different dies, have different heads: those of a die go over the same rows.  dK and dV of a piece, where both are wanted, are workgroups of the
    // same head, and which comes first changes from piece to piece, so that every die gets as many of the longer (8192 tokens, 32 and 8 heads of 128: 1496 us with dK on the dies of even
    // numbers, 1300 ... 1350 so).
    const bool both = g.k_grad && g.v_grad;
    uint32_t head, at = (g.plan ? a.by_heads : a.by_combos).div(g.before + blockIdx.x, head);
    const bool dk = both ? !(__builtin_popcount(at) & 1) : g.k_grad != nullptr;
    if (both) at >>= 1;
    Piece p;
    if (g.plan) {
        if ((int)at >= g.plan->pieces) return;
        p = g.pieces[at];
        if (p.nk == 0) return;
    } else {
        Span s;
        int h;
        uint32_t none;
        if (!place_of<kGradKeys, true>(a, at * a.combos + head, s, h, none)) return;
        head = (uint32_t)h;
        p = Piece{s.q0, s.nq, s.k0, s.nk, s.tile, 0, 0, -1};
        tiles_of_keys(a, p.nq, p.nk, p.tile, H::kKeys, p.from, p.to);
    }
    clear_tiles<H>(smem, 2 * kKeyStage<H>, a.dim);
    if (dk) key_grad<H, true>(g, p, (int)head, smem);
    else key_grad<H, false>(g, p, (int)head, smem);
}

// Gradients of the keys that lie in several parts: a workgroup has 1024 values of one join and head, [keys][2][dim].
template <int DT>
__global__ __launch_bounds__(256) void prompt_grad_join_kernel(PromptGradArgs g, int chunks) {
    const PromptArgs& a = g.p;
    uint32_t head;
    const uint32_t rest = a.by_heads.div(blockIdx.x, head);
    const int join = (int)(rest / (uint32_t)chunks), at = (int)((rest - join * chunks) * 1024 + threadIdx.x * 4);
    if (join >= g.plan->joins) return;
    const KeyJoin j = g.joins[join];
    if (at >= j.keys * 2 * a.dim) return;
    const int64_t pitch = (int64_t)a.kv_heads * kGradKeys * 2 * a.dim;
    const float* from = g.parts + ((int64_t)j.part * a.kv_heads + head) * kGradKeys * 2 * a.dim + at;
    f4 x = {0.f, 0.f, 0.f, 0.f};
    for (int n = 0; n < j.parts; n++) x += *reinterpret_cast<const f4*>(from + n * pitch);
    const int key = at / (2 * a.dim), d = at - key * 2 * a.dim, other = d >= a.dim;
    uint16_t* out = other ? g.k_grad : g.v_grad;
    if (out) store4<DT>(out + ((int64_t)(j.key + key) * a.kv_heads + head) * a.dim + d - other * a.dim, x[0], x[1], x[2], x[3]);
}
