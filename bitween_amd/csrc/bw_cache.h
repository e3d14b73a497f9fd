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
