// bw_prompt_kernel.h - causal attention of many tokens of each sequence, with a window and sinks: what the kernels of the forward and of the gradients
// share, and the forward's.
//
// A workgroup takes a tile of 128 rows of one sequence and one key-value head: a row is a new token and one of the query heads that read the key head, so that
// heads that share keys share their tiles, and a tile spans few tokens, which keeps what the mask cuts off small.  Its four waves have 32 rows each, and the
// keys come by, kKeys at a time, through LDS: two buffers, filled by loads that go from memory to LDS and are waited for a tile later.
//   S^T[key][row] = K Q^T        32 x 32 x 16 MFMAs; A = 32 keys from LDS, B = the wave's rows, in registers
//   P^T = exp2(S^T c - r)        a lane holds row lane % 32, keys 8 j + 4 (lane / 32) + i of each 32
//   O^T[d][row] += V^T P^T       B = P^T as it lies there; A = V^T: transposing reads of the 4 + 4 keys that the lane's half holds
// The order of the keys in an MFMA is free as long as P and V agree, so nothing crosses lanes between the two products.  r is only raised when a score passes
// it by some powers of two (one vote a tile).
//
// LDS: rows of kPitch values; the 16-byte chunk c of row n lies at c ^ swizzle(n), which spreads over all banks both 16 rows at one chunk (K) and 4
// rows at four neighbouring ones (V^T).
//
// What bounds it: the matrix cores and the vector unit of a SIMD, which its two waves share: 32 MFMAs of 32 cycles for a tile of 64 keys and heads of 128, 32 exponentials of 16 cycles and about 130
// other vector instructions of 4; busy 51 % and 46 % of the time, at the clock that the part holds under such load (about 2.1 GHz).  8192 tokens, 32 query and 8 key heads of 128, bfloat16: 510 ... 595 us as
// the clocks of cards differ, and with what ran before, 1079 ... 924 TFLOP/s (the library's product of 8192^3: 1327); 601 us before operands were read ahead of their products, the loop for values that are not finite had become another, and the
// scalars of the loop registers of their own (64 a tile came from spilled vector registers).  Heads of 64: 860 TFLOP/s (the same exponentials for half the products).  Not taken: 32 keys at a time with
// the next scores under the weights (623 us for 564), higher wave priority in either product (nothing), four waves a SIMD with heads of 64 (nine registers in memory, nothing gained).
#pragma once
#include "bw_cache.h"

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));

constexpr int kRows = 128, kWaveRows = 32, kPromptWaves = 4;
// Where weights lie in their 16-bit type: in float16, whose steps end at 2^-24, the largest at 2^12 and more when its reference is set, up to 2^15 until the
// reference is raised; in bfloat16 never above 1, so that no product is larger than its value.  One rounding to the type, at most half a step of a weight (2^-11 of it, 2^-8 in
// bfloat16), as large as the result's own: 1500 tokens with heads of 128 in bfloat16 err by 0.0020 of the result, 0.0016 of which its rounding makes.  A second number for what the rounding
// leaves, and a second product, would take that to 0.0016, and 8192 tokens from 534 to 716 us (heads of 64 162 to 230).
template <int DT> constexpr float kWeightTop = DT == BW_F16 ? 12.f : -8.f;
template <int DT> constexpr float kWeightMost = DT == BW_F16 ? 15.f : 0.f;
constexpr float kLowestScore = -3.4028235e38f;

struct PromptArgs {
    const uint16_t *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    uint16_t* out;                               // [tokens][q_heads][dim]
    float* lse;                                  // [kv_heads][q_tokens * share]: log2 of a row's sum of 2^score, or NULL
    float* partial;                              // parts of rows: see prompt_join_kernel
    const int32_t *q_starts, *k_starts;          // NULL: `sequences` of seq_q and seq_k tokens each
    int q_tokens, k_tokens, sequences, seq_q, seq_k;
    int q_heads, kv_heads, share, dim;
    int window, sinks, splits;
    uint32_t combos, tiles;                      // workgroups: `combos` x (row or key tiles of a sequence, or slots) x splits
    FastDiv by_share, by_combos, by_heads, by_tiles, by_splits;
    float scale;                                 // times log2 e, positive
    uint32_t flip;                               // sign bits that turn the queries for a negative scale
    void set_tiles(uint32_t n) {
        tiles = n;
        by_tiles = FastDiv(n ? n : 1);
    }
    void set_splits(int n) {
        splits = n;
        by_splits = FastDiv((uint32_t)n);
    }
};

// kDim: the head dimension filled up to whole MFMAs; kPitch: values of a row in LDS, a power of two.
template <int DT, int DIM> struct Head {
    static constexpr int kType = DT, kDim = DIM, kPitch = DIM <= 64 ? 64 : DIM <= 128 ? 128 : 256, kSteps = DIM / 16, kBlocks = DIM / 32;
    static constexpr int kKeys = kPitch == 256 ? 32 : 64, kTileBytes = kKeys * kPitch * 2, kChunks = kPitch / 8, kLoadRows = 64 / kChunks;
    static constexpr int kLoads = kTileBytes / 1024 / kPromptWaves;             // of a wave, 64 x 16 bytes each
    static constexpr int kKeyBlocks = kKeys / 32, kResident = kPitch == 256 ? 1 : 2;
};

template <int PITCH> BW_DEV int swizzle(int row) { return PITCH == 64 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : (row & 3) << 2 | (row >> 2 & 3); }

template <int DT> BW_DEV f16v mfma32(u4 a, u4 b, f16v c) {
    if constexpr (DT == BW_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) char lds_char;
BW_DEV uint32_t lds_address(const char* p) { return (uint32_t)(uintptr_t)(const lds_char*)p; }

// 16 bytes (4) of every lane from base + offset to LDS at `to` + 16 (4) lane.  Assembly, because the compiler would wait for it before any read of LDS; the
// waits and barriers are placed by the callers (wait_tiles).  (Wait states: M0 and a scalar that a vector instruction may have written.  M0 is one of the registers that the compiler never
// hands out, which its warning about the list says; naming it keeps its own settings of M0, were there any, from being carried over the statement.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
BW_DEV void load_to_lds(const void* base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(to)) : "memory", "m0");
}
BW_DEV void load4_to_lds(const void* base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(to)) : "memory", "m0");
}
#pragma clang diagnostic pop
// The order of a region's instructions, N of a kind at a time: the compiler reads an operand from LDS right before the product that takes it, and waits for it there.
template <int N> BW_DEV void then_reads() { __builtin_amdgcn_sched_group_barrier(0x100, N, 0); }
template <int N> BW_DEV void then_products() { __builtin_amdgcn_sched_group_barrier(0x008, N, 0); }
template <int N> BW_DEV void then_vector() { __builtin_amdgcn_sched_group_barrier(0x002, N, 0); }
template <int N> BW_DEV void then_exponentials() { __builtin_amdgcn_sched_group_barrier(0x400, N, 0); }
// Nothing is moved past it.
BW_DEV void in_order() { __builtin_amdgcn_sched_barrier(0); }
// N products with PER reads each, AHEAD products' worth of them before the first.
template <int N, int PER, int AHEAD> BW_DEV void reads_ahead() {
    then_reads<PER * (AHEAD < N ? AHEAD : N)>();
    static_for<0, N>([&](auto i) {
        then_products<1>();
        if constexpr (decltype(i)::value + AHEAD < N) then_reads<PER>();
    });
}

// A scalar register of its own for a number that a loop needs: an argument lies in a block of 16, which is read back from a vector register as a whole where there are not enough.
template <class T> BW_DEV T own(T x) {
    asm("" : "+s"(x));
    return x;
}

// What was asked for has arrived, for all waves.
BW_DEV void wait_tiles() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);                          // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// TILES tiles of rows of one head on their way to LDS.  Rows from `rows` on are those of the last one again (the mask hides them); values behind the head's end are not
// loaded.
template <class H, int TILES = 1> struct RowLoader {
    static constexpr int kLoads = H::kLoads * TILES, kKeys = H::kKeys * TILES;
    uint32_t row_bytes, bytes, chunk[kLoads], at;
    int first, whole;                            // row of the lane in the first load; tiles with that many rows are whole ones
    BW_DEV RowLoader(const PromptArgs& a, int lane, int wave, int64_t row) {
        row_bytes = own((uint32_t)(row * 2));
        bytes = own((uint32_t)a.dim * 2);
        whole = own(a.dim == H::kPitch ? kKeys : 0x7fffffff);
        first = wave * kLoads * H::kLoadRows + lane / H::kChunks;
        at = (uint32_t)first * row_bytes;
#pragma unroll
        for (int i = 0; i < kLoads; i++) chunk[i] = (uint32_t)((lane % H::kChunks) ^ swizzle<H::kPitch>(first + i * H::kLoadRows)) * 16;
    }
    BW_DEV void operator()(const void* base, int rows, uint32_t to, int wave) const {
        to += wave * kLoads * 1024;
        if (rows >= whole) {
#pragma unroll
            for (int i = 0; i < kLoads; i++) load_to_lds(base, at + i * H::kLoadRows * row_bytes + chunk[i], to + i * 1024);
        } else {
            uint32_t some = bytes;
            asm("" : "+s"(some));                                // (the comparisons below are not kept in registers over the loop)
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int r = first + i * H::kLoadRows;
                if (chunk[i] < some) load_to_lds(base, (uint32_t)(r < rows ? r : rows - 1) * row_bytes + chunk[i], to + i * 1024);
            }
        }
    }
};

// Operands from a tile in LDS.  rows: 32 of them, step s of 16 values of the head; columns: V^T, 32 values of the head from block m on, 16 of the
// rows in the order 4 h + i, 8 + 4 h + i for half h of the lanes.
template <class H> struct TileReader {
    uint32_t row_at[H::kSteps], column_at[H::kBlocks][2];
    BW_DEV explicit TileReader(int lane) {
        const int n = lane & 31, half = lane >> 5;
#pragma unroll
        for (int s = 0; s < H::kSteps; s++) row_at[s] = (uint32_t)(n * H::kPitch * 2 + ((2 * s + half) ^ swizzle<H::kPitch>(n)) * 16);
        const int i = lane & 15, low = 2 * (lane >> 4 & 1) + (i >> 1 & 1);
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int r = 8 * u + 4 * half + (i >> 2);
                column_at[m][u] = (uint32_t)(r * H::kPitch * 2 + ((4 * m + low) ^ swizzle<H::kPitch>(r)) * 16 + (i & 1) * 8);
            }
    }
    BW_DEV u4 rows(const char* tile, int block, int s) const { return *reinterpret_cast<const u4*>(tile + row_at[s] + block * 32 * H::kPitch * 2); }
    BW_DEV u4 columns(const char* tile, int step, int m) const {
        u2 w[2];
#pragma unroll
        for (int u = 0; u < 2; u++)
            w[u] = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)(tile + column_at[m][u] + step * 16 * H::kPitch * 2)));
        return u4{w[0][0], w[0][1], w[1][0], w[1][1]};
    }
};

template <int DT> constexpr uint32_t kExponent = DT == BW_F16 ? 0x7C00u : 0x7F80u;
template <int DT> BW_DEV bool finite16(uint32_t v) { return (v & kExponent<DT>) != kExponent<DT>; }
// Whether it is true for any thread of the workgroup; through LDS that nothing else is in any more.
template <int WAVES = kPromptWaves> BW_DEV bool any_thread(char* smem, int wave, bool is) {
    const uint64_t hit = __builtin_amdgcn_ballot_w64(is);
    __syncthreads();
    reinterpret_cast<volatile uint32_t*>(smem)[wave] = hit != 0;
    __syncthreads();
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) any |= reinterpret_cast<const uint32_t*>(smem)[i];
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(any);
}
// Infinities and NaN of a tile made 0, by the whole workgroup.
template <class H, int THREADS = 256> BW_DEV void keep_finite(char* tile, int bytes) {
    __syncthreads();
#pragma unroll 1
    for (int at = (int)threadIdx.x * 4; at < bytes; at += THREADS * 4) {
        const uint32_t w = *reinterpret_cast<uint32_t*>(tile + at);
        *reinterpret_cast<uint32_t*>(tile + at) = (finite16<H::kType>(w) ? w & 0xFFFFu : 0u) | (finite16<H::kType>(w >> 16) ? w & 0xFFFF0000u : 0u);
    }
    __syncthreads();
}
// What keep_finite takes out of a tile's transposed product: an infinity or a NaN in row n goes into the sums of those for which seen(n) is true, and no others.
template <class H, class Seen> BW_DEV void add_nonfinite(const char* tile, int rows, int lane, f16v* acc, Seen&& seen) {
    const int half = lane >> 5;
#pragma unroll 1
    for (int n = 0; n < rows; n++) {
        const char* row = tile + n * H::kPitch * 2;
        bool any = false;
#pragma unroll
        for (int w = 0; w < (H::kPitch + 127) / 128; w++) {
            const int at = (lane + 64 * w) * 4;
            const uint32_t v = at < H::kPitch * 2 ? *reinterpret_cast<const uint32_t*>(row + at) : 0u;
            any |= !finite16<H::kType>(v) || !finite16<H::kType>(v >> 16);
        }
        if (!__builtin_amdgcn_ballot_w64(any)) continue;
        const bool sees = seen(n);
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int c = (4 * m + b) ^ swizzle<H::kPitch>(n);
                const u2 v = *reinterpret_cast<const u2*>(row + c * 16 + half * 8);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t x = v[i / 2] >> (16 * (i & 1)) & 0xFFFFu;
                    if (sees && !finite16<H::kType>(x)) acc[m][4 * b + i] += widen16<H::kType>((uint16_t)x);
                }
            }
    }
}

// A sequence's new tokens q0 ... q0 + nq - 1 and all its tokens k0 ... k0 + nk - 1, of which the new ones are the last; `tile` of its tiles of rows or of keys.
struct Span { int q0, nq, k0, nk, tile; };

BW_DEV int start_at(const int32_t* starts, int i, int all) {
    const int s = starts[i];
    return s < 0 ? 0 : s < all ? s : all;
}
// The tokens of sequence s; s = sequences: those behind the last one, sequences + 1: those before the first, which have no keys (or no rows).
BW_DEV void tokens_at(const int32_t* starts, int s, int sequences, int all, int& from, int& count) {
    from = s <= sequences ? start_at(starts, s, all) : 0;
    const int to = s < sequences ? start_at(starts, s + 1, all) : s == sequences ? all : start_at(starts, 0, all);
    count = to > from ? to - from : 0;
}
// The slot'th tile over all sequences, TILE rows or keys each; false: there are fewer.  The last tile of a sequence, which sees the most, goes first (rows), or
// the first, which most see (keys).
template <int TILE, bool KEYS> BW_DEV bool find_tile(const PromptArgs& a, uint32_t slot, Span& p) {
    const int lane = (int)threadIdx.x & 63;
    uint32_t before = 0;
    for (int base = 0; base < a.sequences + 2; base += 64) {
        const int s = base + lane;
        uint32_t mine = 0;
        if (s < a.sequences + 2) {
            int from, count;
            tokens_at(KEYS ? a.k_starts : a.q_starts, s, a.sequences, KEYS ? a.k_tokens : a.q_tokens, from, count);
            mine = ((uint32_t)count * (KEYS ? 1u : (uint32_t)a.share) + TILE - 1) / TILE;
        }
        uint32_t sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t other = __shfl_up(sum, o, 64);
            if (lane >= o) sum += other;
        }
        const uint64_t hit = __builtin_amdgcn_ballot_w64(slot >= before + sum - mine && slot < before + sum);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            const uint32_t first = before + __builtin_amdgcn_readlane(sum - mine, at), count = __builtin_amdgcn_readlane(mine, at);
            const int found = base + at;
            p.tile = (int)(slot - first);
            if (!KEYS) p.tile = (int)count - 1 - p.tile;
            tokens_at(a.q_starts, found, a.sequences, a.q_tokens, p.q0, p.nq);
            tokens_at(a.k_starts, found, a.sequences, a.k_tokens, p.k0, p.nk);
            if (found >= a.sequences) (KEYS ? p.nq : p.nk) = 0;
            p.q0 = __builtin_amdgcn_readfirstlane(p.q0);
            p.nq = __builtin_amdgcn_readfirstlane(p.nq);
            p.k0 = __builtin_amdgcn_readfirstlane(p.k0);
            p.nk = __builtin_amdgcn_readfirstlane(p.nk);
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// What this workgroup has: a tile of one sequence and one key-value head.  Neighbouring workgroups have different heads (and go to different dies), so that the
// tiles of a head, which read the same keys, share a die's cache wherever 8 divides the number of heads.
template <int TILE, bool KEYS> BW_DEV bool place_of(const PromptArgs& a, uint32_t block, Span& p, int& head, uint32_t& split) {
    uint32_t combo;
    uint32_t slot = a.by_combos.div(block, combo);
    split = a.by_tiles.div(slot, slot);
    if (a.q_starts) {
        head = (int)combo;
        return find_tile<TILE, KEYS>(a, slot, p);
    }
    uint32_t h;
    const uint32_t s = a.by_heads.div(combo, h);
    head = (int)h;
    p = Span{(int)s * a.seq_q, a.seq_q, (int)s * a.seq_k, a.seq_k, (int)(KEYS ? slot : a.tiles - 1 - slot)};
    return true;
}

// The tiles of keys that rows at positions `low` ... `high` see, `tile` keys each: `sinks` first ones, then from `first` on, `count` in all.
struct KeyTiles {
    int sinks, first, count;
    BW_DEV KeyTiles(const PromptArgs& a, int low, int high, int nk, int tile) {
        if (high < 0 || nk <= 0) { sinks = first = count = 0; return; }
        const int from = low - a.window + 1;
        first = from > 0 ? from / tile : 0;
        const int s = a.sinks < nk ? a.sinks : nk;
        sinks = (s + tile - 1) / tile;
        if (sinks > first) sinks = first;
        const int last = high / tile;
        count = sinks + last - first + 1;
    }
    BW_DEV int operator[](int i) const { return i < sinks ? i : i - sinks + first; }
    // The split'th of a.splits parts.
    BW_DEV void part(const PromptArgs& a, uint32_t split, int& from, int& to) const {
        uint32_t rest;
        const int each = (int)a.by_splits.div((uint32_t)(count + a.splits - 1), rest);
        from = (int)split * each < count ? (int)split * each : count;
        to = from + each < count ? from + each : count;
    }
};
// Keys and values of the tiles one after the other: what the next one's rows begin at.
template <class H, int TILES = 1> struct KeyWalk {
    static constexpr int kKeys = H::kKeys * TILES;
    const char *k, *v;
    uint32_t k_step, v_step;
    int at, i, jump_at, jump;
    BW_DEV KeyWalk(const PromptArgs& a, const Span& p, int head, const KeyTiles& tiles, int begin) {
        i = begin;
        at = tiles[begin] * kKeys;
        jump_at = own(tiles.sinks);
        jump = own(tiles.first - tiles.sinks + 1);
        k_step = own((uint32_t)(kKeys * 2 * a.k_row));        // (rows are 2^24 - 1 apart at most)
        v_step = own((uint32_t)(kKeys * 2 * a.v_row));
        k = own((const char*)(a.k + (int64_t)(p.k0 + at) * a.k_row + head * a.k_head));
        v = own((const char*)(a.v + (int64_t)(p.k0 + at) * a.v_row + head * a.v_head));
    }
    BW_DEV void step() {
        const int by = ++i == jump_at ? jump : 1;
        at += by * kKeys;
        k += (uint64_t)k_step * (uint32_t)by;
        v += (uint64_t)v_step * (uint32_t)by;
    }
};

// Which keys rows at positions low ... high see of N from `at` on: none, all, or without those that are later than some row, or that some row's window has left.
enum Seen { kNone = -1, kAll = 0, kLater = 1, kLeft = 2 };
template <int N> struct SeenOf {
    int none_above, all_to, window_from, sinks, all_from;
    BW_DEV SeenOf(const PromptArgs& a, int low, int high, bool any) {
        none_above = own(any ? high : -1);                       // (no rows: nothing is seen)
        all_to = own(low - N + 1);
        window_from = own(low - a.window + 1 - N);
        sinks = own(a.sinks);
        all_from = own(high - a.window + 1);
    }
    BW_DEV int operator()(int at) const {
        if (at > none_above || (at <= window_from && at >= sinks)) return kNone;
        return (at > all_to ? kLater : 0) | (at < all_from && at + N > sinks ? kLeft : 0);
    }
};
// Values of a lane, for keys from + 8 (j / 4) + j % 4 and a row at `position`: `hidden` in place of those that the row does not see.
template <int N> BW_DEV void hide(int which, const PromptArgs& a, int position, int from, float hidden, float* x) {
    if (which & kLater) {
        const int last = position - from;
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = 8 * (j / 4) + j % 4 <= last ? x[j] : hidden;
    }
    if (which & kLeft) {
        const int left = position - a.window - from, sinks = a.sinks - from;
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = 8 * (j / 4) + j % 4 > left || 8 * (j / 4) + j % 4 < sinks ? x[j] : hidden;
    }
}
BW_DEV bool sees(const PromptArgs& a, int position, int key) { return key <= position && (key > position - a.window || key < a.sinks); }

// 16 bytes of a row for every step of 16 values of the head, zeros where there is nothing: an operand of the wave's rows.
template <class H> BW_DEV void load_row(u4* out, const uint16_t* row, bool live, int dim, int half) {
#pragma unroll
    for (int s = 0; s < H::kSteps; s++) {
        const int d = 16 * s + 8 * half;
        out[s] = live && d < dim ? *reinterpret_cast<const u4*>(row + d) : u4{0, 0, 0, 0};
    }
}

// sum + the two 16-bit values of a word
template <int DT> BW_DEV float add_pair(uint32_t w, float sum) {
    typedef __bf16 b2v __attribute__((ext_vector_type(2)));
    if constexpr (DT == BW_BF16) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2v, w), __builtin_bit_cast(b2v, 0x3F803F80u), sum, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), __builtin_bit_cast(h2, 0x3C003C00u), sum, false);
}

// The rows of a wave: lane l (and l + 32) has row first + l of the sequence.
struct Row {
    int token, head, position;                   // of the sequence's new tokens; of the key head's query heads
    bool live;
    BW_DEV Row(const PromptArgs& a, const Span& p, int row) {
        live = row < p.nq * a.share;
        uint32_t rest;
        token = (int)a.by_share.div((uint32_t)(live ? row : 0), rest);
        head = (int)rest;
        position = p.nk - p.nq + token;
    }
};
// Positions of rows from ... to - 1 of a sequence (the last one that there is, at most).
BW_DEV void positions_of(const PromptArgs& a, const Span& p, int from, int to, int& low, int& high) {
    uint32_t rest;
    const int last = to < p.nq * a.share ? to - 1 : p.nq * a.share - 1;
    low = p.nk - p.nq + (int)a.by_share.div((uint32_t)from, rest);
    high = p.nk - p.nq + (int)a.by_share.div((uint32_t)(last > from ? last : from), rest);
}

// Four values d ... d + 3 of an output row.
template <int DT> BW_DEV void store4(uint16_t* p, float x, float y, float z, float w) { *reinterpret_cast<u2*>(p) = u2{narrow_pair<DT>(x, y), narrow_pair<DT>(z, w)}; }

// Whether a sum of the lane is an infinity or a NaN.
template <int BLOCKS> BW_DEV bool not_finite(const f16v* acc) {
    float check = 0.f;
#pragma unroll
    for (int m = 0; m < BLOCKS; m++)
#pragma unroll
        for (int j = 0; j < 16; j++) check = __builtin_fmaf(acc[m][j], 0.f, check);
    return check != 0.f;
}

template <class H> BW_DEV void clear_tiles(char* smem, int bytes, int dim) {
    if (dim == H::kPitch) return;                                // (values behind the head's end are not loaded)
    for (int i = (int)threadIdx.x * 16; i < bytes; i += 256 * 16) *reinterpret_cast<u4*>(smem + i) = u4{0, 0, 0, 0};
    __syncthreads();
}

// GROUPS 2: half the rows to a workgroup, and two tiles of keys at a time, of which two waves have one each; what they sum for a row is added up at the end, through LDS.  Half the steps,
// where there are few workgroups and their steps, one after the other, are what it takes (512 tokens, 32 heads of 128: 17.9 us, 13.0 so; with many workgroups the steps overlap without: 2048 tokens, 32 and 8 heads, 54.8, 71.6 so).
template <class H, int GROUPS>
__global__ __launch_bounds__(256, H::kResident) void prompt_forward_kernel(PromptArgs a) {
    extern __shared__ __align__(1024) char smem[];               // [2][K, V]
    constexpr int kTileRows = kRows / GROUPS, kBytes = H::kTileBytes * GROUPS;
    constexpr int DT = H::kType;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5;
    Span p;
    int head;
    uint32_t split;
    if (!place_of<kTileRows, false>(a, blockIdx.x, p, head, split)) return;
    clear_tiles<H>(smem, 4 * kBytes, a.dim);
    const int group = wave / (kPromptWaves / GROUPS), row0 = p.tile * kTileRows + wave % (kPromptWaves / GROUPS) * kWaveRows, rows = p.nq * a.share;
    const Row row(a, p, row0 + (lane & 31));
    const int64_t token = p.q0 + row.token;
    u4 q[H::kSteps];
    load_row<H>(q, a.q + token * a.q_row + (head * a.share + row.head) * a.q_head, row.live, a.dim, half);
#pragma unroll
    for (int s = 0; s < H::kSteps; s++)
#pragma unroll
        for (int j = 0; j < 4; j++) q[s][j] ^= a.flip;

    int low, high, wave_low, wave_high;
    positions_of(a, p, p.tile * kTileRows, (p.tile + 1) * kTileRows, low, high);
    positions_of(a, p, row0 < rows ? row0 : p.tile * kTileRows, row0 + kWaveRows, wave_low, wave_high);
    const KeyTiles tiles(a, low, high, p.nk, H::kKeys * GROUPS);
    int begin, end;
    tiles.part(a, split, begin, end);

    const RowLoader<H, GROUPS> load_k(a, lane, wave, a.k_row), load_v(a, lane, wave, a.v_row);
    const TileReader<H> read(lane);
    const SeenOf<H::kKeys> seen(a, wave_low, wave_high, row0 < rows);
    const uint32_t lds = own(lds_address(smem));
    const int keys = own(p.nk);
    const float scale = own(a.scale);
    auto fetch = [&](const KeyWalk<H, GROUPS>& next) __attribute__((always_inline)) {
        const uint32_t to = lds + (next.i & 1) * 2 * kBytes;
        load_k(next.k, keys - next.at, to, wave);
        load_v(next.v, keys - next.at, to + kBytes, wave);
    };

    f16v acc[H::kBlocks];
    float r, l;
    // An infinity or a NaN among the values leaves nothing finite in 0 times it, also where the mask hides its token.  Where a result is not finite, the tile
    // is done again, carefully: the products take finite values only, the others are added to the rows that see them.  (A loop of its own: what it needs is not there in the other.)
    auto pass = [&](auto is_careful) __attribute__((always_inline)) {
        constexpr bool careful = decltype(is_careful)::value;
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++) acc[m] = f16v{};
        r = kLowestScore;
        l = 0.f;
        KeyWalk<H, GROUPS> next(a, p, head, tiles, begin);
        if (begin < end) fetch(next);
        for (int i = begin; i < end; i++) {
            const int at = next.at + group * H::kKeys;
            next.step();
            wait_tiles();
            if (next.i < end) fetch(next);
            char *stage = smem + (i & 1) * 2 * kBytes, *tile = stage + group * H::kTileBytes, *values = tile + kBytes;
            const int which = seen(at);
            if constexpr (careful) {
                if (which != kNone) add_nonfinite<H>(values, H::kKeys, lane, acc, [&](int n) { return sees(a, row.position, at + n); });
                keep_finite<H>(stage + kBytes, kBytes);
            }
            if (which == kNone) continue;
            f16v s[H::kKeyBlocks];
#pragma unroll
            for (int b = 0; b < H::kKeyBlocks; b++) s[b] = f16v{};
#pragma unroll
            for (int k = 0; k < H::kSteps; k++)
#pragma unroll
                for (int b = 0; b < H::kKeyBlocks; b++) s[b] = mfma32<DT>(read.rows(tile, b, k), q[k], s[b]);
            reads_ahead<H::kKeyBlocks * H::kSteps, 1, 4>();
            in_order();
            u4 v[H::kBlocks];
#pragma unroll
            for (int m = 0; m < H::kBlocks; m++) v[m] = read.columns(values, 0, m);
            if (which != kAll) {
#pragma unroll
                for (int b = 0; b < H::kKeyBlocks; b++) hide<16>(which, a, row.position, at + 32 * b + 4 * half, -INFINITY, reinterpret_cast<float*>(&s[b]));
            }
            float tops[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
            for (int b = 0; b < H::kKeyBlocks; b++)
#pragma unroll
                for (int j = b ? 0 : 4; j < 16; j++) tops[j / 4] = fmaxf(tops[j / 4], s[b][j]);
            float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            top *= scale;
            if (__builtin_amdgcn_ballot_w64(top > r + kWeightMost<DT>)) {
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                // (of those rows only that need it: a row's result does not hang on its neighbours)
                const float raised = top > r + kWeightMost<DT> ? top - kWeightTop<DT> : r, keep = raised == r ? 1.f : __builtin_amdgcn_exp2f(r - raised);
                r = raised;
                l *= keep;
#pragma unroll
                for (int m = 0; m < H::kBlocks; m++) acc[m] *= keep;
            }
            // 16 keys at a time: their values and weights are got ready while the products of the 16 before them are under way
            auto weights = [&](int step) __attribute__((always_inline)) {
                u4 w;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int n = 8 * (step & 1) + 2 * j;
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[step / 2][n], scale, -r)), y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[step / 2][n + 1], scale, -r));
                    w[j] = narrow_pair<DT>(x, y);
                }
                return w;
            };
            u4 w = weights(0);
#pragma unroll
            for (int step = 0; step < 2 * H::kKeyBlocks; step++) {
                u4 next_v[H::kBlocks], next_w;
                if (step + 1 < 2 * H::kKeyBlocks) {
#pragma unroll
                    for (int m = 0; m < H::kBlocks; m++) next_v[m] = read.columns(values, step + 1, m);
                    next_w = weights(step + 1);
                }
                // (the sum of the weights as they are multiplied, two at a time: what their rounding adds to the values it takes off again)
#pragma unroll
                for (int j = 0; j < 4; j++) l = add_pair<DT>(w[j], l);
#pragma unroll
                for (int m = 0; m < H::kBlocks; m++) acc[m] = mfma32<DT>(v[m], w, acc[m]);
                if (step + 1 < 2 * H::kKeyBlocks) {
                    then_reads<2 * H::kBlocks>();
                    static_for<0, H::kBlocks>([&](auto) {
                        then_products<1>();
                        then_vector<(16 + H::kBlocks - 1) / H::kBlocks>();
                        then_exponentials<(8 + H::kBlocks - 1) / H::kBlocks>();
                    });
                    w = next_w;
#pragma unroll
                    for (int m = 0; m < H::kBlocks; m++) v[m] = next_v[m];
                }
                in_order();
            }
        }
    };
    pass(std::false_type{});
    if (any_thread(smem, wave, row.live && not_finite<H::kBlocks>(acc))) pass(std::true_type{});

    l += __shfl_xor(l, 32, 64);
    if constexpr (GROUPS > 1) {
        static_assert(GROUPS == 2, "two");
        char* other = smem + wave % 2 * (H::kBlocks * 4096 + 512);
        __syncthreads();
        if (group) {
#pragma unroll
            for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
                for (int b = 0; b < 4; b++) *reinterpret_cast<f4*>(other + ((4 * m + b) * 64 + lane) * 16) = f4{acc[m][4 * b], acc[m][4 * b + 1], acc[m][4 * b + 2], acc[m][4 * b + 3]};
            reinterpret_cast<float*>(other + H::kBlocks * 4096)[lane] = r;
            reinterpret_cast<float*>(other + H::kBlocks * 4096)[64 + lane] = l;
        }
        __syncthreads();
        if (group) return;
        const float r2 = reinterpret_cast<float*>(other + H::kBlocks * 4096)[lane], l2 = reinterpret_cast<float*>(other + H::kBlocks * 4096)[64 + lane];
        const float top = fmaxf(r, r2), f1 = __builtin_amdgcn_exp2f(r - top), f2 = __builtin_amdgcn_exp2f(r2 - top);
        r = top;
        l = l * f1 + l2 * f2;
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const f4 x = *reinterpret_cast<const f4*>(other + ((4 * m + b) * 64 + lane) * 16);
#pragma unroll
                for (int i = 0; i < 4; i++) acc[m][4 * b + i] = acc[m][4 * b + i] * f1 + x[i] * f2;
            }
    }
    if (!row.live) return;
    const int64_t index = (int64_t)head * a.q_tokens * a.share + token * a.share + row.head;       // of the row among all
    const bool empty = row.position < 0 || p.nk == 0;             // no key is seen: zeros
    if (a.splits > 1) {                                           // (see prompt_join_kernel)
        const int64_t parts = (int64_t)a.q_tokens * a.q_heads * a.splits, at = index * a.splits + split;
        // (a row that sees no key has none in this part either, also where other rows of its tile do: it is empty, not a row whose scores are all minus infinity)
        const float reference = begin < end && !empty ? r : -INFINITY;
        if (half == 0) reinterpret_cast<u2*>(a.partial)[at] = u2{__builtin_bit_cast(uint32_t, reference), __builtin_bit_cast(uint32_t, l)};
        float* part = a.partial + parts * 2 + at * a.dim;
#pragma unroll
        for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int d = 32 * m + 8 * b + 4 * half;
                if (d < a.dim) *reinterpret_cast<f4*>(part + d) = f4{acc[m][4 * b], acc[m][4 * b + 1], acc[m][4 * b + 2], acc[m][4 * b + 3]};
            }
        return;
    }
    const float inv = empty ? 0.f : 1.f / l;
    if (a.lse && half == 0) a.lse[index] = empty ? INFINITY : r + __builtin_amdgcn_logf(l);
    uint16_t* out = a.out + (token * a.q_heads + head * a.share + row.head) * a.dim;
#pragma unroll
    for (int m = 0; m < H::kBlocks; m++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int d = 32 * m + 8 * b + 4 * half;
            if (d < a.dim) store4<DT>(out + d, acc[m][4 * b] * inv, acc[m][4 * b + 1] * inv, acc[m][4 * b + 2] * inv, acc[m][4 * b + 3] * inv);
        }
}
