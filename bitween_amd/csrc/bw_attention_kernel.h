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
    float scale;                                 // times log2 e
};

// A value that all lanes read at one address, through the scalar cache: lengths and table, which nothing writes while the kernel runs.
BW_DEV int32_t uniform_load(const int32_t* p, int64_t i) { return ((const __attribute__((address_space(4))) int32_t*)p)[i]; }

BW_DEV int clipped(const AttentionArgs& a, int n) { return n < 0 ? 0 : n < a.max_tokens ? n : a.max_tokens; }
BW_DEV int tokens_of(const AttentionArgs& a, uint32_t b) { return clipped(a, uniform_load(a.lengths, b)); }
BW_DEV uint32_t tiles_of(int tokens) { return ((uint32_t)tokens + kTile - 1) >> kTileShift; }
BW_DEV uint32_t units_of(int tokens) { return tokens ? tiles_of(tokens) + kSegmentCost : 0; }

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
template <class Wanted>
BW_DEV Place find_sequence(const AttentionArgs& a, uint32_t* lds, Wanted&& wanted) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const bool wide = a.B > 64;
    const int run = wide ? (a.B + 255) >> 8 : 1, first = wide ? (int)threadIdx.x * run : lane;
    uint32_t mine = 0;
    for (int b = first; b < first + run && b < a.B; b++) mine += units_of(clipped(a, a.lengths[b]));
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
        const uint32_t t = run == 1 ? mine : units_of(clipped(a, a.lengths[b]));
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
    const int32_t* table;
};
BW_DEV Segment segment_of(const AttentionArgs& a, uint32_t b, uint32_t hq, uint32_t at, uint32_t left) {
    Segment g;
    g.b = b;
    g.hq = hq;
    g.n = tokens_of(a, b);
    g.tiles = tiles_of(g.n);
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
        left = tiles_of(tokens_of(a, b)) + kSegmentCost;
    } else {
        const Place place = find_sequence(a, lds, [&](uint32_t all, uint32_t before, uint32_t units) {
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
        const uint32_t units = units_of(tokens_of(a, b));
        hq = rest / units;
        at = rest - hq * units;
    }
    Segment g = segment_of(a, b, hq, at, left);
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
    auto halves_of = [&](const Segment& g, uint32_t t) {
        const int at = (int)t * kTile;
        Halves h;
        h.page[0] = (uint32_t)uniform_load(g.table, at >> a.page_shift);
        h.page[1] = at + 16 < g.n ? (uint32_t)uniform_load(g.table, (at + 16) >> a.page_shift) : 0xFFFFFFFFu;
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
            const uint32_t t = g.from + wave + i * kWaves;
            if (t >= g.to) break;
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
            after = segment_of(a, b, hq, 0, left);
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
        auto step = [&](Tile<F>& tile, const uint32_t t) __attribute__((always_inline)) {
            // The second half of the workgroups shares its CUs with the first, whose waves, being older, go before: 17 against 21 us of a launch's 24.
            // Going first every other tile evens it out (48 sequences of up to 8192 tokens, 8 heads of 128 in 8 bits: 46.2 against 47.4 us).
            __builtin_amdgcn_s_setprio(0);
            if (blockIdx.x >= gridDim.x / 2 && (t / kWaves & 1)) __builtin_amdgcn_s_setprio(1);
            const uint32_t next = t + kAhead * kWaves;
            const bool more = next < to;
            Halves hn = {};
            if (more) hn = halves_of(g, next);
            // Tokens that do not count: behind the end, or on a page outside the cache.
            const bool full = (int)t * kTile + kTile <= n && tile.h.page[0] < a.pages && tile.h.page[1] < a.pages;
            const Halves h = tile.h;
            any |= h.page[0] < a.pages || h.page[1] < a.pages;
            auto counts = [&](int half, int i) { return (int)t * kTile + 16 * half + 4 * kg + i < n && h.page[half] < a.pages; };
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
}
