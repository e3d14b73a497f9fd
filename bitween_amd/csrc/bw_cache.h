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
    if (c->pages >= (int64_t)1 << 31 || c->kv_heads > 65535) return BW_EUNSUPPORTED;
    if (!bw_aligned(c->keys, 16) || !bw_aligned(c->values, 16)) return BW_EALIGN;
    return BW_OK;
}

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
template <int DT> BW_DEV uint16_t narrow16(float f) {
    if constexpr (DT == BW_F16) return __builtin_bit_cast(uint16_t, (_Float16)f);
    else return f32_to_bf16(f);
}
BW_DEV float f16_bits(uint32_t u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)u); }
