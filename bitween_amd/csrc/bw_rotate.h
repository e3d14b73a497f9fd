// bw_rotate.h - what the kernels that rotate heads (bw_rotate.hip, bw_append.hip) share: which values a thread has, the angles of its pairs, sums over a head.
//
// A thread owns CH values of a head and the CH values half a rotation further on, the pairs that turn together (behind the rotated part:
// twice CH neighbours), so that a pair never leaves its thread.  2^lane_shift neighbouring threads hold a head (as many as it needs, filled up
// to a power of two), and the sums that the norm needs go over them with cross-lane moves.
#pragma once
#include "bw_cache.h"

constexpr int kMaxDim = 256;

struct RotateArgs {
    const uint16_t *q, *k, *gq, *gk;
    int64_t q_row, q_head, k_row, k_head, gq_row, gq_head, gk_row, gk_head;
    uint16_t *q_out, *k_out;                     // rotated heads, or the gradients of the inputs
    const float *cos, *sin;
    const int64_t* positions;
    const void *q_weight, *k_weight;
    float* partial;                              // [blocks][dim]: sums of dw, the queries' blocks first
    int64_t table_rows;
    int T, q_heads, k_heads, dim, half, lanes, lane_shift, weight_f32;
    int q_blocks;                                // gradient: blocks that serve the queries
    float eps;
    int axes;                                    // positions of a token: [axes][position_pitch]
    int64_t position_pitch;
    uint32_t axis[8];                            // of each pair, two bits
    uint32_t slices, k_slices;                   // threads (of a head's place) for each token: see slices_of; gradient: the queries' and the keys'
};

// CH 16-bit values as they come from memory, and as float32.
template <int CH> using Raw = std::conditional_t<CH == 8, u4, u2>;
template <int CH> BW_DEV Raw<CH> load_raw(const uint16_t* p) { return *reinterpret_cast<const Raw<CH>*>(p); }
template <int DT, int CH> BW_DEV void widen_raw(const Raw<CH>& w, float* x) {
#pragma unroll
    for (int j = 0; j < CH; j++) x[j] = widen16<DT>((uint16_t)(w[j / 2] >> (16 * (j & 1))));
}

template <int DT, int CH>
BW_DEV void store_chunk(uint16_t* p, const float* x) {
    uint32_t w[CH / 2];
#pragma unroll
    for (int j = 0; j < CH / 2; j++) w[j] = narrow_pair<DT>(x[2 * j], x[2 * j + 1]);
    if constexpr (CH == 8) *reinterpret_cast<u4*>(p) = u4{w[0], w[1], w[2], w[3]};
    else *reinterpret_cast<u2*>(p) = u2{w[0], w[1]};
}

template <int DT, int CH>
BW_DEV void load_weight(const void* w, int f32, int at, float* x) {
    if (f32) {
#pragma unroll
        for (int j = 0; j < CH; j++) x[j] = ((const float*)w)[at + j];
    } else {
        widen_raw<DT, CH>(load_raw<CH>((const uint16_t*)w + at), x);
    }
}

template <int CH>
BW_DEV void load_floats(const float* p, float* x) {
#pragma unroll
    for (int j = 0; j < CH / 4; j++) {
        const f4 v = *reinterpret_cast<const f4*>(p + 4 * j);
        x[4 * j] = v[0]; x[4 * j + 1] = v[1]; x[4 * j + 2] = v[2]; x[4 * j + 3] = v[3];
    }
}

// The two chunks of lane c of a head, and whether they turn.
template <int CH>
BW_DEV void chunks_of(const RotateArgs& a, int c, int& first, int& second, bool& turns) {
    const int pairs = a.half / CH;
    turns = c < pairs;
    first = turns ? c * CH : 2 * a.half + 2 * (c - pairs) * CH;
    second = turns ? first + a.half : first + CH;
}

// Over the 2^shift lanes of a head, each with the sum: neighbours, pairs, then mirrored halves of 8 and of 16, whose lanes hold the same by then.
template <int CTRL> BW_DEV float from_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
BW_DEV float head_sum(float v, int shift) {
    if (shift > 0) v += from_lane<0xB1>(v);
    if (shift > 1) v += from_lane<0x4E>(v);
    if (shift > 2) v += from_lane<0x141>(v);
    if (shift > 3) v += from_lane<0x140>(v);
    if (shift > 4) v += __shfl_xor(v, 16, 64);
    return v;
}

// Where a token is: one position, or (AXES) up to four, of which each pair has its own.  Padding, if one of them lies outside the table.
template <bool AXES> struct Position {
    int64_t at[AXES ? 4 : 1];
    bool kept;
    BW_DEV Position(const RotateArgs& a, int token) {
#pragma unroll
        for (int i = 0; i < (AXES ? 4 : 1); i++) at[i] = a.positions[AXES && i < a.axes ? i * a.position_pitch + token : token];
        kept = at[0] >= 0 && at[0] < a.table_rows;
        if constexpr (AXES) {
#pragma unroll
            for (int i = 1; i < 4; i++) kept &= i >= a.axes || (at[i] >= 0 && at[i] < a.table_rows);
        }
    }
};

// cos and sin of a thread's pairs.
template <int CH> struct Angle {
    float c[CH], s[CH];
    BW_DEV void load(const RotateArgs& a, const Position<false>& p, int first) {
        load_floats<CH>(a.cos + p.at[0] * a.half + first, c);
        load_floats<CH>(a.sin + p.at[0] * a.half + first, s);
    }
    // The rows of those axes that a pair of the thread has; where they lie one behind the other, nearly every thread has one.
    BW_DEV void load(const RotateArgs& a, const Position<true>& p, int first) {
        const uint32_t axis = a.axis[first / 16] >> (first % 16 * 2);
        float x[4][CH], y[4][CH];
        bool has[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            has[i] = false;
#pragma unroll
            for (int j = 0; j < CH; j++) has[i] |= (axis >> 2 * j & 3) == (uint32_t)i;
            if (i < a.axes && has[i]) {
                load_floats<CH>(a.cos + p.at[i] * a.half + first, x[i]);
                load_floats<CH>(a.sin + p.at[i] * a.half + first, y[i]);
            }
        }
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const uint32_t n = axis >> 2 * j & 3;
            c[j] = n == 0 ? x[0][j] : n == 1 ? x[1][j] : n == 2 ? x[2][j] : x[3][j];
            s[j] = n == 0 ? y[0][j] : n == 1 ? y[1][j] : n == 2 ? y[2][j] : y[3][j];
        }
    }
    // SIGN 1: turned by the angle, -1: turned back
    template <int SIGN> BW_DEV void turn(float* x, float* y) const {
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const float u = x[j], v = y[j];
            x[j] = u * c[j] - SIGN * v * s[j];
            y[j] = v * c[j] + SIGN * u * s[j];
        }
    }
};

// Values of a chunk: 8, where whole 16-byte chunks fill the rotated halves and what lies behind them.
static inline int chunk_of(const bw_heads* h) { return h->dim % 16 == 0 && h->rotary % 16 == 0 ? 8 : 4; }

static inline int heads_check(const bw_heads* h, int act_dtype) {
    if (!h || h->tokens < 0 || h->q_heads < 1 || h->k_heads < 1 || h->dim < 1 || h->rotary < 1 || h->rotary > h->dim || h->table_rows < 1) return BW_EINVAL;
    if (h->tokens > 0 && (!h->cos || !h->sin || !h->positions)) return BW_EINVAL;
    if (act_dtype != BW_F16 && act_dtype != BW_BF16) return BW_EUNSUPPORTED;
    if ((h->q_weight || h->k_weight) && h->weight_dtype != act_dtype && h->weight_dtype != BW_F32) return BW_EUNSUPPORTED;
    if (h->dim % 8 || h->rotary % 8 || h->dim > kMaxDim) return BW_EUNSUPPORTED;
    if (h->q_heads > 65535 || h->k_heads > 65535 || h->tokens >= (int64_t)1 << 31) return BW_EUNSUPPORTED;
    const int64_t items = h->tokens * ((int64_t)h->q_heads + h->k_heads);
    if (items >= (int64_t)1 << 31 || items * h->dim >= (int64_t)1 << 36) return BW_EUNSUPPORTED;
    if (!bw_aligned(h->cos, 16) || !bw_aligned(h->sin, 16) || !bw_aligned(h->positions, 8) || !bw_aligned(h->q_weight, 16) || !bw_aligned(h->k_weight, 16))
        return BW_EALIGN;
    return BW_OK;
}

static inline RotateArgs rotate_args(const bw_heads* h, const bw_axes* x = nullptr) {
    RotateArgs a = {};
    a.cos = h->cos; a.sin = h->sin;
    a.positions = h->positions;
    a.q_weight = h->q_weight; a.k_weight = h->k_weight;
    a.weight_f32 = h->weight_dtype == BW_F32;
    a.table_rows = h->table_rows;
    a.T = (int)h->tokens;
    a.q_heads = h->q_heads; a.k_heads = h->k_heads;
    a.dim = h->dim;
    a.half = h->rotary / 2;
    a.lanes = h->dim / (2 * chunk_of(h));
    a.lane_shift = bw_log2(a.lanes);
    a.eps = h->eps;
    a.axes = x ? x->count : 1;
    a.position_pitch = h->tokens;
    if (x) {
        int in_order = 0, axis = 0;
        for (int i = 0; i < a.half; i++) {
            while (axis < x->count && in_order >= x->sections[axis]) { axis++; in_order = 0; }
            in_order++;
            const int turn = i % x->count, of = x->interleaved ? (i < x->count * x->sections[turn] ? turn : 0) : axis;
            a.axis[i / 16] |= (uint32_t)of << (i % 16 * 2);
        }
    }
    return a;
}

// Threads (of one place in a head) for each token, of which each has as many of its `heads` as leave the chip about 1024 workgroups, 8 at most, and their angles once: 16384 tokens
// of 32 and 8 heads of 128 and three axes 111 us with one head each, 73 so.
static inline int slices_of(const RotateArgs& a, int heads) {
    const int64_t rounds = ((int64_t)a.T * heads << a.lane_shift) / (256 * 1024);
    const int each = (int)(rounds < 1 ? 1 : rounds < 8 ? rounds : 8);
    return (heads + each - 1) / each;
}

// The axes fit the pairs: they take all of them, and interleaved ones find theirs.
static inline int axes_check(const bw_axes* x, int rotary) {
    if (!x || x->count < 1 || x->count > 4) return BW_EINVAL;
    int64_t all = 0;
    for (int i = 0; i < x->count; i++) {
        if (x->sections[i] < 0) return BW_EINVAL;
        all += x->sections[i];
        if (x->interleaved && i && x->sections[i] > 0 && ((int64_t)x->sections[i] - 1) * x->count + i >= rotary / 2) return BW_EINVAL;
    }
    return all == rotary / 2 ? BW_OK : BW_EINVAL;
}

