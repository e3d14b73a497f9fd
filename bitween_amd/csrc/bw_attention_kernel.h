// bw_attention_kernel.h - attention of one new token over a paged cache: the kernel template, its arguments and the split of its work.
//
// Work is counted in tiles of 32 tokens of one segment: one sequence, one key-value head, up to 16 of the query heads that read it.  A segment
// counts as its tiles and kSegmentCost more, what beginning and joining it takes.  The segments, one after the other, are cut into equal pieces,
// one for each workgroup, so that sequences of very different length load the chip evenly; lengths are read on the GPU, so the cut
// follows them.  A segment that lies in one piece is finished by its workgroup; the parts of one that lies in several go to the workspace
// and are joined by attention_join_kernel.
//
// The four waves of a workgroup take tiles in turn, each with a running reference r and sum l of its own.  One wave, one tile, everything in
// registers:
//   S^T[token][query] = K Q^T        A = 16 tokens of K (a lane: token lane % 16, 8 values of the head at a time), B = 16 queries
//   P^T = exp2(S^T c - r)            a lane holds query lane % 16, tokens 4 (lane / 16) + i of each half of the tile
//   O^T[d][query] += V^T P^T         B = P^T as it lies there; A = V^T: a lane loads a piece of the rows of just those 8 tokens and pairs
//                                    the tokens with byte permutes
// The order of the head's values in an MFMA is free as long as K and Q agree, and that of the tokens as long as P and V agree, so between the two
// products nothing crosses lanes, and there is no LDS before the waves are joined.  r is only raised when a score passes it by some powers of two (one vote
// a tile, shuffles where it is raised).  Over codes pairs, weights and narrow pieces of V go from lane to lane in registers (DPP), see Fold and Exchange.
//
// P enters as 16-bit numbers, each rounded to nearest, whose sum it is: three in bfloat16, which hold all of a float32 (two, cut to 16 bits, gave every
// 170th result of the largest case another bfloat16 neighbour than the exact value's, where float32 weights give every 1500th; three cost 0 ... 2 %), two in
// float16.  Its steps end at 2^-24, so r is kept where the largest P is 2^12 ... 2^15: a weight errs by 2^-22 of itself or 2^-37 of the largest.  (With
// the largest at 1 ... 2^8, and cut instead of rounded, 8192 weights e^-14 of one more came out 0.9 % low.)
//
// Fewer than 16 queries leave columns of the MFMAs empty: the matrix cores have room (16 KB of a 16-bit tile take 24 MFMAs in float16, 32 in
// bfloat16, 400 and 500 cycles of one SIMD, and about 6000 cycles of a SIMD's share of HBM).
//
// Codes enter the MFMAs as they are: a whole number in the low bits of a 16-bit float is that number times 2^-24, a subnormal, which the matrix cores
// take, so that unpacking is a byte permute or a shift and an AND for two codes.  They line products up as if a subnormal were 2^-14 and cut them
// 24 bits below the largest: 2^-16 of a code's unit (measured: sums of 32 within 5e-4 units of the largest factor), nothing beside 255
// units, but too much beside 15, so 4-bit codes go in four bits higher, where it is 2^-20.
// Scales and zero points are applied in float32:
//   K: S = s (Q . c - z sum Q) for each group
//   V: O += (P s) c, and another MFMA whose rows are the zero points sums (P s) z, which is taken off at the end
// so no value is rounded on its way in.  What enters, P s, can be anything from 2^-24 to 2^16 times P, and a head's groups may be that far apart, so
// every group has a power of two of its own for every query, its reach: P s times it is 2^12 ... 2^15 at its largest too, and the group's sums are
// divided by it at the end.  P itself stays float32, and so do r and l.  (With one reference for all groups of a token a group 2^-10 of the largest
// erred by 2^-10.  The reach and its vote for each group cost 1 ... 4 % with heads of 128, 9 % with 16 queries over groups of 32 in 8 bits, 18 % with four groups
// of 64 to a head.)
//
// Over a window (window_kernel, the same body): a segment's tiles are those of its sinks and those from the window's first token on, and only where a tile's tokens do not all count is each looked at.
// One sequence of 131072 tokens that sees 4096 and 4 sinks, 32 and 8 heads of 128, 16 bits: 9.9 us and 3.4 for the join (17 MB, 3.3 us: latency); 48 sequences that see 2000 in 8 bits: 38 and 4.7 us
// (185 MB, 4.9 TB/s); 128 that see 500, 12 heads of 64 in 4 bits: 24 us (48 MB: the issue of instructions, as without a window).
#pragma once
#include "bw_cache.h"

constexpr int kTile = 32, kTileShift = 5, kWaves = 4, kQueries = 16;
// Tiles that beginning and joining a segment is worth: with 2 the pieces of many short segments are waited for (32 sequences of up to 1000 tokens, 8 heads of
// 128 in 8 bits: 29.4 us; 5: 23.7; 8 and 12: 20.4), with 12 the long ones (64 of up to 8192 in 16 bits: 166.4 against 165.2 with 8 and 163.3 with 2).
constexpr uint32_t kSegmentCost = 8;
BW_DEV uint32_t many_units(int queries) { return queries > 8 ? 16 : 6; }          // see split_of
// Where weights lie in their 16-bit type: the largest at 2^kTop and more when its reference is set, up to 2^kMost until the reference is raised.  In
// bfloat16, whose steps have no end but whose values reach 2^128, never above 1: the products are no larger than the values.
template <bool BF16> constexpr int kTop = BF16 ? -8 : 12;
template <bool BF16> constexpr int kMost = BF16 ? 0 : 15;
// Over codes P itself stays float32 and may pass its reference by 2^8; a group's reach begins at 2^100.
constexpr float kSlack = 8.f;
constexpr int kFirstReach = 100;
// The reference before any finite score: a score of minus infinity lies as far below it as below any other, and weighs 0.  A wave that has met no token
// hands on minus infinity instead.
constexpr float kLowest = -3.4028235e38f;

// A segment that begins in a workgroup's piece (in its second slot) and goes on in the first slots of the next parts - 1 pieces; parts 0: none.
struct alignas(16) Joint { uint32_t b, hq, parts; };          // (what lies behind them in the workspace begins at 16 bytes)

struct AttentionArgs {
    const uint16_t* q;
    int64_t q_row, q_head;
    const int32_t *table, *lengths;
    int64_t table_row;
    const uint8_t *keys, *values;
    const uint32_t *key_meta, *value_meta;
    uint16_t* out;
    Joint* joints;                               // what each workgroup leaves to join
    float* partial;                              // 2 slots for each workgroup: r [16], l [16], O [queries][dim]
    uint32_t pages;
    int B, q_heads, kv_heads, share, queries, q_groups;   // queries: of a segment, at most 16; q_groups: segments of a key-value head
    int dim, row_bytes, page_shift, max_tokens, q_bf16, cus, whole;
    int window, sinks;                           // the last `window` tokens count, and the first `sinks`
    float scale;                                 // times log2 e
};

// A value that all lanes read at one address, through the scalar cache: lengths and table, which nothing writes while the kernel runs.
BW_DEV int32_t uniform_load(const int32_t* p, int64_t i) { return ((const __attribute__((address_space(4))) int32_t*)p)[i]; }

BW_DEV int clipped(const AttentionArgs& a, int n) { return n < 0 ? 0 : n < a.max_tokens ? n : a.max_tokens; }
BW_DEV int tokens_of(const AttentionArgs& a, uint32_t b) { return clipped(a, uniform_load(a.lengths, b)); }
BW_DEV uint32_t tiles_of(int tokens) { return ((uint32_t)tokens + kTile - 1) >> kTileShift; }
// What counts of n tokens: the sinks and those from `from` on, in `tiles` tiles, the first `sinks` of which come before `skip` ones that are left out.
struct Visible { int from; uint32_t sinks, skip, tiles; };
template <bool WINDOW> BW_DEV Visible visible_of(const AttentionArgs& a, int n) {
    if constexpr (!WINDOW) return {0, 0, 0, tiles_of(n)};
    Visible v = {n > a.window ? n - a.window : 0, 0, 0, tiles_of(n)};
    if (v.from <= a.sinks) v.from = 0;
    const uint32_t first = (uint32_t)v.from >> kTileShift, sinks = tiles_of(a.sinks);
    v.sinks = sinks < first ? sinks : first;
    v.skip = first - v.sinks;
    v.tiles -= v.skip;
    return v;
}
template <bool WINDOW> BW_DEV uint32_t units_of(const AttentionArgs& a, int tokens) { return tokens ? visible_of<WINDOW>(a, tokens).tiles + kSegmentCost : 0; }

// The pieces, in units: `longer` of them have one more than the others.  Tile i of a segment is its unit kSegmentCost + i.
struct Split {
    uint32_t pieces, size, longer;
    BW_DEV uint32_t start(uint32_t w) const { return w * size + (w < longer ? w : longer); }
    BW_DEV uint32_t piece_of(uint32_t unit) const {
        const uint32_t head = longer * (size + 1);
        return unit < head ? unit / (size + 1) : longer + (unit - head) / size;
    }
};
// Less than many_units for every workgroup that can be resident: one piece for a CU at most, of so many units that its waves have equally many.
// Smaller ones cost more in parts to join, the more the queries of each, and a second piece on some of the CUs is waited for by all.  8 sequences of
// 8192, 16 queries of one head of 128: 14.8 us in 176 pieces against 17.8 in 512; 4 of 1024, 8 heads with 8 queries: 11.4 in 160, 12.9 in 256 of 5 units;
// 16 of 8192 with 16 queries of one head (8 units for each of 512): 19.5 in 212, 20.8 in 512.  4 sequences of 4096, 8 heads with 4 queries in 8 bits
// (8.5 units): 17.7 in 242, 15.9 in 512; one of 2048, 32 heads in 8 bits (4.5 units): 13.8 in 192, 13.0 in 512, but 4 of 2000 with 16 queries 16.4 and 17.3.
BW_DEV Split split_of(const AttentionArgs& a, uint32_t units, uint32_t grid) {
    const uint32_t total = units * (uint32_t)(a.kv_heads * a.q_groups), round = (uint32_t)(a.cus * kWaves);
    const uint32_t size = (total + round - 1) / round * kWaves, pieces = total >= grid * many_units(a.queries) ? grid : size ? (total + size - 1) / size : 0;
    Split s = {};
    s.pieces = pieces < grid ? pieces : grid;
    s.size = s.pieces ? total / s.pieces : 0;
    s.longer = total - s.pieces * s.size;
    return s;
}

// A sequence, the units (for one head) of the sequences before it, and of all.
struct Place { uint32_t b, before, all; };

// The sequence that wanted(all, before, units) picks, by sums over the sequences.  Up to 64 sequences every wave does it for itself, a lane for
// each sequence; more: thread i sums a run of them, the runs are added up over the lanes and then the four waves.
template <bool WINDOW, class Wanted>
BW_DEV Place find_sequence(const AttentionArgs& a, uint32_t* lds, Wanted&& wanted) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const bool wide = a.B > 64;
    const int run = wide ? (a.B + 255) >> 8 : 1, first = wide ? (int)threadIdx.x * run : lane;
    uint32_t mine = 0;
    for (int b = first; b < first + run && b < a.B; b++) mine += units_of<WINDOW>(a, clipped(a, a.lengths[b]));
    uint32_t sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t other = __shfl_up(sum, o, 64);
        if (lane >= o) sum += other;
    }
    Place p = {0, 0, 0};
    if (!wide) {
        p.all = __builtin_amdgcn_readlane(sum, 63);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(lane < a.B && wanted(p.all, sum - mine, mine));
        if (hit) {
            p.b = (uint32_t)__builtin_ctzll(hit);
            p.before = __builtin_amdgcn_readlane(sum - mine, p.b);
        }
        return p;
    }
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    uint32_t before = sum - mine;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        const uint32_t part = __builtin_amdgcn_readfirstlane(lds[w]);
        if (w < wave) before += part;
        p.all += part;
    }
    for (int b = first; b < first + run && b < a.B; b++) {
        const uint32_t t = run == 1 ? mine : units_of<WINDOW>(a, clipped(a, a.lengths[b]));
        if (wanted(p.all, before, t)) {
            lds[4] = (uint32_t)b;
            lds[5] = before;
        }
        before += t;
    }
    __syncthreads();
    p.b = __builtin_amdgcn_readfirstlane(lds[4]);
    p.before = __builtin_amdgcn_readfirstlane(lds[5]);
    return p;
}

BW_DEV void store_out(const AttentionArgs& a, int64_t row, int d, f4 o) {
    const uint2 w = a.q_bf16 ? uint2{narrow_pair<BW_BF16>(o[0], o[1]), narrow_pair<BW_BF16>(o[2], o[3])} : uint2{narrow_pair<BW_F16>(o[0], o[1]), narrow_pair<BW_F16>(o[2], o[3])};
    *reinterpret_cast<uint2*>(a.out + row * a.dim + d) = w;
}

// ---- formats ----
// How the values of a head lie in MFMAs: NK operand blocks of 32 values for K and Q, NV output blocks of 16 values for V.
//   K, Q: lane group kg = lane / 16 holds values k_at(block, kg) .. + 7      V: lane m = lane % 16 holds value v_at(m, j) for block j

typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// 16 bits, DT = BW_F16 | BW_BF16; DP: the head dimension filled up to 64, 128 or 256.  Lanes behind the head's end read its beginning again:
// against zeros of Q, and into outputs that nobody stores.
template <int DT, int DP> struct Format16 {
    static constexpr bool kCodes = false, kBf16 = DT == BW_BF16;
    static constexpr int kBits = 16, kPerV = DP / 16;
    static constexpr int kDim = DP, NK = DP / 32, NV = DP / 16, kGroups = 1, kKeyWords = NK * 4, kValueWords = NV / 2, kValueLoads = (DP + 127) / 128, kMerge = 1;
    static BW_DEV int k_at(int block, int kg) { return 32 * block + 8 * kg; }
    // 64: 4 neighbouring values (8 bytes) of a lane; 128: 8 (16 bytes); 256: 8 of each half
    static BW_DEV int v_at(int m, int j) { return DP == 64 ? 4 * m + j : (j >> 3) * 128 + 8 * m + (j & 7); }
};
// BITS-bit codes in GROUPS groups of GS values: every MFMA, of K and of V, keeps to one group.
template <int BITS, int GROUPS, int GS> struct FormatQ {
    static constexpr bool kCodes = true, kBf16 = false;
    static constexpr int kBits = BITS, kGroup = GS, kGroups = GROUPS, kDim = GROUPS * GS, NK = kDim / 32, NV = kDim / 16;
    static constexpr int kPerK = GS / 32, kPerV = GS / 16;                  // operand blocks and output blocks of a group
    static constexpr int kKeyGroupWords = GS * BITS / 128, kKeyWords = GROUPS * kKeyGroupWords;
    // A lane's part of a group in a row of V is kValueBytes; parts of less than a word are loaded kMerge groups at a time (see exchanged)
    static constexpr int kGroupBytes = GS * BITS / 8, kValueBytes = kPerV * BITS / 8, kMerge = kValueBytes < 4 ? 4 / kValueBytes : 1;
    static constexpr int kValueGroupWords = kValueBytes > 4 ? kValueBytes / 4 : 1, kMerged = GROUPS / kMerge, kValueLoads = kMerged + GROUPS % kMerge, kValueWords = kValueGroupWords * kValueLoads;
    static constexpr int value_word(int c, int j) { return kMerge == 1 ? c * kValueGroupWords + j * BITS / 32 : c < kMerged * kMerge ? c / kMerge : c - kMerged * (kMerge - 1); }
    static constexpr int value_code(int c, int j) { return kMerge == 1 ? j % (32 / BITS) : (c < kMerged * kMerge ? c % kMerge * kPerV : 0) + j; }
    static BW_DEV int k_at(int block, int kg) { return (block / kPerK) * GS + kg * (GS / 4) + (block % kPerK) * 8; }
    static BW_DEV int v_at(int m, int j) { return (j / kPerV) * GS + m * kPerV + j % kPerV; }
};

template <bool BF16> BW_DEV f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// Two float32 as 16-bit numbers, to nearest; split_pair leaves in x and y what is missing (exactly).
template <bool BF16> BW_DEV uint32_t pair_of(float x, float y) { return narrow_pair<BF16 ? BW_BF16 : BW_F16>(x, y); }
template <bool BF16> BW_DEV uint32_t split_pair(float& x, float& y) {
    const uint32_t p = pair_of<BF16>(x, y);
    if constexpr (BF16) {
        x -= __builtin_bit_cast(float, p << 16);
        y -= __builtin_bit_cast(float, p & 0xFFFF0000u);
    } else {
        x -= (float)as_h2(p)[0];
        y -= (float)as_h2(p)[1];
    }
    return p;
}

// Codes of one word as operand pairs, in units of 2^-kUnit.  8 bits: (0, 1) (2, 3); 4 bits: (0, 4) (1, 5) (2, 6) (3, 7), the order of Q too.
template <int BITS> constexpr int kUnit = BITS == 8 ? 24 : 20;
template <int BITS> BW_DEV void key_codes(uint32_t w, uint32_t* out) {
    if constexpr (BITS == 8) {
        out[0] = __builtin_amdgcn_perm(0u, w, 0x0C010C00u);
        out[1] = __builtin_amdgcn_perm(0u, w, 0x0C030C02u);
    } else {
        out[0] = w << 4 & 0x00F000F0u;
        out[1] = w & 0x00F000F0u;
        out[2] = w >> 4 & 0x00F000F0u;
        out[3] = w >> 8 & 0x00F000F0u;
    }
}
template <int BITS> BW_DEV int query_order(int e) { return BITS == 4 ? (e >> 1) + 4 * (e & 1) : e; }

// 16 bits of each of two tokens' words, and code J of both as an operand pair.
template <bool HIGH> BW_DEV uint32_t token_pair(uint32_t second, uint32_t first) { return __builtin_amdgcn_perm(second, first, HIGH ? 0x07060302u : 0x05040100u); }
template <int BITS, int J> BW_DEV uint32_t value_codes(uint32_t second, uint32_t first) {
    if constexpr (BITS == 8) {
        return __builtin_amdgcn_perm(second, first, 0x0C040C00u + 0x00010001u * (J % 4));
    } else {
        const uint32_t a = token_pair<(J / 4) % 2 != 0>(second, first);
        return (J % 4 == 0 ? a << 4 : a >> 4 * (J % 4 - 1)) & 0x00F000F0u;
    }
}

// Where a tile's two halves lie: pages as the table names them.
struct Halves { uint32_t page[2]; };

// One tile's rows and pairs as they come from memory.
template <class F> struct Tile {
    Halves h;
    uint32_t key[2][F::kKeyWords];
    uint32_t value[8][F::kValueWords];           // token 4 kg + i of half h: 4 h + i
    uint32_t pairs[2][F::kGroups];               // of a group: see Fold
};
// What lane L of the 16, and of the 4, has.
template <int L> BW_DEV uint32_t row_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x150 + L, 0xF, 0xF, true); }
template <int L> BW_DEV uint32_t quad_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, L * 0x55, 0xF, 0xF, true); }
// What the lane N further on (of 16, around) has.
template <int N> BW_DEV uint32_t lane_after(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x120 + 16 - N, 0xF, 0xF, true); }

// Groups whose part for a lane is 1 or 2 bytes of a row of V: instead of that from each, lane m loads word m / MERGE of group m % MERGE, and the MERGE lanes of
// one word index exchange their bytes or halves, so that each has its part of every group in one register.
// Groups of 32, 8 heads of 128: 102 against 169 us with 4 queries each (64 sequences of up to 8192 tokens), 68 against 98 with 16 (32 sequences);
// 8 bits 127 against 175 and 91 against 111.
template <int MERGE> struct Exchange {
    uint32_t pairs, quads;                       // byte selectors
    BW_DEV explicit Exchange(int m) : pairs(m & 1 ? 0x03070105u : 0x06020400u), quads(m & (MERGE / 2) ? 0x03020706u : 0x05040100u) {}
    BW_DEV uint32_t operator()(uint32_t v) const {
        if constexpr (MERGE == 4) v = __builtin_amdgcn_perm((uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true), v, pairs);
        return __builtin_amdgcn_perm((uint32_t)__builtin_amdgcn_mov_dpp((int)v, MERGE == 4 ? 0x4E : 0xB1, 0xF, 0xF, true), v, quads);
    }
};

// Few queries leave columns of the MFMAs empty, and with them most of what a lane does between the two products: over codes that is more than the
// unpacking.  With 8 or fewer queries (FOLD 2) or 4 (FOLD 4) they are there 2 or 4 times, and the lanes of each copy ("part" m / (16 / FOLD)) take only
// their share of the tile's tokens, kTokens = 8 / FOLD instead of 8 each; the weights go back to the first copy's lanes for the second product.
// 64 sequences of up to 8192 tokens, 8 heads of 128, groups of 32, 4 queries: 102 against 113 us in 4 bits, 127 against 152 us in 8 (fewer registers go
// to memory, too); groups of 128: no difference; one sequence of 65537: 27.0 against 28.2.
//   token j of part p is token 4 h + i of the lane's 8: FOLD 1: j;  2: h = p, i = j;  4: h = p / 2, i = 2 (p % 2) + j
//   a group's pairs, one load for all: FOLD 1: lanes 0 ... 7 the keys' 8 tokens, 8 ... 15 the values';  2: lanes 4 c + i of part p the keys' and, in a
//   second register, the values' token j = i;  4: lanes 0, 1 of the four of part p the keys' tokens, 2, 3 the values'
template <int FOLD> struct Fold {
    static constexpr int kTokens = 8 / FOLD, kColumns = 16 / FOLD, kRegisters = FOLD == 2 ? 2 : 1;
    int part;
    bool odd, high;                              // of part
    BW_DEV explicit Fold(int m) : part(m / kColumns), odd(part & 1), high(FOLD == 4 ? part & 2 : part & 1) {}
    BW_DEV int token(int j) const { return FOLD == 1 ? j : FOLD == 2 ? 4 * part + j : 2 * part + j; }          // 4 h + i
    BW_DEV int pair_token(int m) const { return FOLD == 1 ? m & 7 : FOLD == 2 ? 4 * part + (m & 3) : 2 * part + (m & 1); }
    static BW_DEV bool pair_is_value(int m) { return FOLD == 1 ? m & 8 : m & 2; }                              // (FOLD 2: by register)
    static BW_DEV float select(bool which, float yes, float no) { return which ? yes : no; }      // (its operands are there: no branch)
    template <int J> BW_DEV float pick(const f4* d) const {                                                   // of the products of both halves
        if constexpr (FOLD == 1) return d[J >> 2][J & 3];
        if constexpr (FOLD == 2) return select(high, d[1][J], d[0][J]);
        return select(high, select(odd, d[1][(2 + J) & 3], d[1][J & 3]), select(odd, d[0][(2 + J) & 3], d[0][J & 3]));
    }
    template <int J> static BW_DEV uint32_t key_pair(uint32_t first) {
        if constexpr (FOLD == 1) return row_lane<J>(first);
        else return quad_lane<J>(first);
    }
    template <int J> static BW_DEV uint32_t value_pair(uint32_t first, uint32_t second) {
        if constexpr (FOLD == 1) return row_lane<8 + J>(first);
        else if constexpr (FOLD == 2) return quad_lane<J>(second);
        else return quad_lane<2 + J>(first);
    }
    // zero points of tokens 2 i and 2 i + 1, side by side
    template <int I> static BW_DEV uint32_t zero_pair(uint32_t both) { return row_lane<FOLD == 1 ? 8 + 2 * I : FOLD == 2 ? 8 * (I >> 1) + 2 * (I & 1) : 4 * I + 2>(both); }
    // the lane's weights (pairs of tokens) to those of all 8
    static BW_DEV u4 all(const uint32_t* own) {
        if constexpr (FOLD == 1) return u4{own[0], own[1], own[2], own[3]};
        else if constexpr (FOLD == 2) return u4{own[0], own[1], lane_after<8>(own[0]), lane_after<8>(own[1])};
        else return u4{own[0], lane_after<4>(own[0]), lane_after<8>(own[0]), lane_after<12>(own[0])};
    }
    // over the parts
    static BW_DEV float max(float v) {
        if constexpr (FOLD == 4) v = fmaxf(v, __shfl_xor(v, 4, 64));
        if constexpr (FOLD >= 2) v = fmaxf(v, __shfl_xor(v, 8, 64));
        return v;
    }
    static BW_DEV float sum(float v) {
        if constexpr (FOLD == 4) v += __shfl_xor(v, 4, 64);
        if constexpr (FOLD >= 2) v += __shfl_xor(v, 8, 64);
        return v;
    }
};

template <int WORDS, bool NT = false> BW_DEV void load_words(const uint8_t* p, uint32_t* out) {
    if constexpr (WORDS % 4 == 0) {
#pragma unroll
        for (int i = 0; i < WORDS / 4; i++) {
            const u4 v = NT ? __builtin_nontemporal_load(reinterpret_cast<const u4*>(p) + i) : reinterpret_cast<const u4*>(p)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) out[4 * i + j] = v[j];
        }
    } else if constexpr (WORDS == 2) {
        const u2 v = NT ? __builtin_nontemporal_load(reinterpret_cast<const u2*>(p)) : *reinterpret_cast<const u2*>(p);
        out[0] = v[0];
        out[1] = v[1];
    } else {
        static_assert(WORDS == 1, "words of a lane");
        out[0] = NT ? __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p)) : *reinterpret_cast<const uint32_t*>(p);
    }
}

// Values are read past the caches, which leaves those to the keys, whose cache lines are taken by more than one load: 165 against 182 us at 64 sequences
// of up to 8192 16-bit tokens (8 heads of 128), 96 against 106 us in 8 bits, the keys too no further use.  Not with 64 values to a head, whose loads
// of values share lines as well: 15.2 against 16.1 us at 128 sequences of 512.
template <class F> constexpr bool kPast = F::kDim > 64;

// Workgroups of a CU at a time, as the registers allow: 27.7 us with three against 33.6 with two at 64 sequences of 2048 tokens of 12 heads of 64 in 8 bits.
// Three for heads of 128 leave too few for groups of 32 (175 against 118 us in 4 bits) and won 4 % over groups of 128, nothing in 8 bits.
constexpr int resident_workgroups(int dim) { return dim > 128 ? 1 : dim > 64 ? 2 : 3; }

// Tiles that a wave has asked for.  Two where the registers hold them: 74.3 us against 75.6 at 64 sequences of up to 8192 tokens, 8 heads of 128, 4 bits in
// groups of 128, 102 against 104 in groups of 32; with more of them in registers (8 or more queries) 67 us became 74, and 8 and 16 bits, whose
// tiles are larger, gain nothing or lose.
template <class F, int FOLD> constexpr int tiles_ahead = F::kBits == 4 && F::kDim <= 128 && (F::kGroups <= 2 || FOLD == 4) ? 2 : 1;

// What a workgroup has of a segment: tiles from ... to - 1 of `tiles`.
struct Segment {
    uint32_t b, hq, from, to, tiles, units;      // units: of the piece that it takes
    int n, head, q_head, queries;
    Visible seen;
    const int32_t* table;
    BW_DEV uint32_t place(uint32_t t) const { return t < seen.sinks ? t : t + seen.skip; }          // of tile t among all of the sequence's
};
template <bool WINDOW> BW_DEV Segment segment_of(const AttentionArgs& a, uint32_t b, uint32_t hq, uint32_t at, uint32_t left) {
    Segment g;
    g.b = b;
    g.hq = hq;
    g.n = tokens_of(a, b);
    g.seen = visible_of<WINDOW>(a, g.n);
    g.tiles = g.seen.tiles;
    const uint32_t all = g.tiles + kSegmentCost, end = left < all - at ? at + left : all;
    g.from = at > kSegmentCost ? at - kSegmentCost : 0;
    g.to = end > kSegmentCost ? end - kSegmentCost : 0;
    g.units = end - at;
    g.head = (int)(hq / (uint32_t)a.q_groups);
    const int first_query = (int)(hq - (uint32_t)g.head * a.q_groups) * kQueries;
    g.queries = a.share - first_query < kQueries ? a.share - first_query : kQueries;
    g.q_head = g.head * a.share + first_query;
    g.table = a.table + (int64_t)b * a.table_row;
    return g;
}

template <class F, int FOLD>
__global__ __launch_bounds__(256, resident_workgroups(F::kDim)) void attention_kernel(AttentionArgs a) {
    constexpr bool WINDOW = false;
#include "bw_attention_body.h"
}
template <class F, int FOLD>
__global__ __launch_bounds__(256, resident_workgroups(F::kDim)) void window_kernel(AttentionArgs a) {
    constexpr bool WINDOW = true;
#include "bw_attention_body.h"
}

template <class F, int FOLD> static void launch_attention(const AttentionArgs& a, uint32_t grid, hipStream_t stream) {
    if (a.window < a.max_tokens) hipLaunchKernelGGL((window_kernel<F, FOLD>), dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attention_kernel<F, FOLD>), dim3(grid), dim3(256), 0, stream, a);
}
