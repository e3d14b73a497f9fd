// bw_cache.h - what the kernels around the key-value cache (bw_cache.hip, bw_attention.hip) share.
#pragma once
#include "bw_common.h"

// What every entry point asks of a cache; page_size is a power of two, so that a token's page and row are a shift and a mask.
static inline int bw_cache_check(const bw_cache* c) {
    if (!c || !c->keys || !c->values || c->pages < 1 || c->kv_heads < 1 || c->page_size < 1 || c->dim < 1) return BW_EINVAL;
    if (c->bits != 16 && c->bits != 8 && c->bits != 4) return c->bits == 2 ? BW_EUNSUPPORTED : BW_EINVAL;
    if (c->bits == 16) {
        if (c->dtype != BW_F16 && c->dtype != BW_BF16) return BW_EUNSUPPORTED;
    } else {
        if (!c->key_meta || !c->value_meta || c->group < 1 || c->dim % c->group) return BW_EINVAL;
        if (c->group != 32 && c->group != 64 && c->group != 128) return BW_EUNSUPPORTED;
        if (!bw_aligned(c->key_meta, 16) || !bw_aligned(c->value_meta, 16)) return BW_EALIGN;
    }
    if (c->dim % 8 || c->dim > 256 || c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) return BW_EUNSUPPORTED;
    if (c->pages >= (int64_t)1 << 31 || c->kv_heads > 65535 || c->pages * c->page_size * c->kv_heads >= (int64_t)1 << 53) return BW_EUNSUPPORTED;
    if (!bw_aligned(c->keys, 16) || !bw_aligned(c->values, 16)) return BW_EALIGN;
    return BW_OK;
}

// n / d and what is left for n < 2^31, by one multiplication.
struct FastDiv {
    uint32_t d, mul;
    int shift;
    FastDiv(uint32_t divisor = 1) : d(divisor), mul(0), shift(0) {
        if (d == 1) return;                                   // mul 0: n itself
        int bits = 1;
        while ((1ull << bits) < d) bits++;
        mul = (uint32_t)((1ull << (31 + bits)) / d + 1);
        shift = bits - 1;
    }
    BW_DEV uint32_t div(uint32_t n, uint32_t& rest) const {
        const uint32_t q = mul ? __umulhi(n, mul) >> shift : n;
        rest = n - q * d;
        return q;
    }
};

static inline int bw_log2(int v) {
    int s = 0;
    while ((1 << s) < v) s++;
    return s;
}

// 16-bit value of either type as float32, and back (round to nearest even).
template <int DT> BW_DEV float widen16(uint16_t u) {
    if constexpr (DT == BW_F16) return (float)__builtin_bit_cast(_Float16, u);
    else return bf16_to_f32(u);
}
template <int DT> BW_DEV uint32_t narrow_pair(float x, float y) {
    if constexpr (DT == BW_F16) return as_u32(h2{(_Float16)x, (_Float16)y});
    else {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, b2{(__bf16)x, (__bf16)y});        // (one instruction)
    }
}
template <int DT> BW_DEV uint16_t narrow16(float f) { return (uint16_t)narrow_pair<DT>(f, f); }
BW_DEV float f16_bits(uint32_t u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)u); }

// ---- quantisation of a group of a head's values ----
//
// The code of x is rint(x / s) of the exact quotient: with r = 1 / s to within a unit of its last place, t = x r and one step t + (x - t s) r the
// result is the correctly rounded quotient wherever rint could tell a difference - x has at most 11 significant bits and s 11, so a
// quotient up to 256 that is not exactly half way between two whole numbers lies at least 2^-13 from half way, and one that is half way has at
// most 10 bits, which the step returns exactly (the residual is exact in the fused operation).  The range over 15 or 255 is that step too, with the
// correctly rounded reciprocal: the correctly rounded quotient (checked over a whole binade and samples of all others).
//
// Extrema of 16-bit floats are whole-number maxima of their bits: a positive value's bits grow with it, a negative one's are negative, so
// max(0, bits) over a group is its largest value (or 0), max(0, bits ^ sign) its most negative one, and an infinity or a NaN shows as bits from the
// infinity's on.  Both fit one register on the way over the lanes.

// Larger of the two 16-bit whole numbers of each half.
typedef short s2 __attribute__((ext_vector_type(2)));
BW_DEV uint32_t max16(uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s2, a), __builtin_bit_cast(s2, b))); }
// Of N words of two 16-bit values: low half the largest value (0, if that is more), high half the size of the most negative one.
template <int N> BW_DEV uint32_t extrema_of(const uint32_t* w) {
    uint32_t hi = 0, lo = 0;
#pragma unroll
    for (int j = 0; j < N; j++) {
        hi = max16(hi, w[j]);
        lo = max16(lo, w[j] ^ 0x80008000u);
    }
    return max16(__builtin_amdgcn_perm(lo, hi, 0x05040100u), __builtin_amdgcn_perm(lo, hi, 0x07060302u));
}

// Scale and zero point of a group with these extrema, and the codes of its values.
template <int DT, int BITS> struct GroupCoder {
    // 1.5 2^23 added: the nearest whole number (ties to even) in the low bits, and whole numbers may be added to it
    static constexpr float kTop = (float)((1 << BITS) - 1), kWhole = 12582912.f;
    float s, r, z;
    uint32_t pair;                               // as it is stored
    BW_DEV float whole(float v) const {
        const float t = v * r;
        return __builtin_fmaf(__builtin_fmaf(-t, s, v), r, t) + kWhole;
    }
    BW_DEV explicit GroupCoder(uint32_t both) {
        constexpr float inv_top = 1.f / kTop;
        constexpr uint32_t inf = DT == BW_F16 ? 0x7C00u : 0x7F80u;
        const bool bad = (both & 0xFFFFu) >= inf || (both >> 16) >= inf;
        const float largest = widen16<DT>((uint16_t)both), smallest = -widen16<DT>((uint16_t)(both >> 16));
        // the scale rounds up, so that no code has to be clipped for its rounding; never 0
        const float range = largest - smallest, t0 = range * inv_top;
        const float step = fminf(__builtin_fmaf(__builtin_fmaf(-t0, kTop, range), inv_top, t0), 65504.f);
        uint32_t sb = __builtin_bit_cast(uint16_t, (_Float16)step);
        sb += f16_bits(sb) < step ? 1 : 0;
        sb = sb ? sb : 1;
        s = f16_bits(sb);
        r = __builtin_amdgcn_rcpf(s);
        z = fminf(whole(-smallest) - kWhole, kTop);
        pair = (bad ? 0x7E00u : sb) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)z) << 16;
    }
    // the code's bits, with others above them (a group with a NaN is marked by its scale)
    BW_DEV uint32_t code(float x) const { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_fmed3f(whole(x) + z, kWhole, kWhole + kTop)); }
};
// The low bytes of four words.
BW_DEV uint32_t bytes_of(uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b3, b2, 0x0C0C0400u), __builtin_amdgcn_perm(b1, b0, 0x0C0C0400u), 0x05040100u);
}

// Two pieces of memory of `bytes` that share some.
static inline bool bw_overlap(const void* a, const void* b, int64_t bytes) {
    const int64_t apart = (int64_t)((const char*)a - (const char*)b);
    return apart < bytes && apart > -bytes;
}
