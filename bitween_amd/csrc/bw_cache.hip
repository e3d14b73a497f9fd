// Writing tokens into the paged key-value cache, quantised as they are written, and reading them back.
//
// A thread owns 8 consecutive values of one token's key or value head: 16 bytes of 16-bit input, and 16, 8 or 4 bytes of the cache.
// The group / 8 neighbouring threads of a group agree on its extrema with cross-lane shuffles (group / 8 divides 64 and every row starts at
// a multiple of it, so a group never leaves its wave), and the first of them stores the group's pair.
//
// The code of x is rint(x / s) of the exact quotient: with r = fl(1 / s), t = fl(x r) and one step t + (x - t s) r the result is the
// correctly rounded quotient wherever rint could tell a difference - x has at most 11 significant bits and s 11, so a quotient up to 256
// that is not exactly half way between two whole numbers lies at least 2^-13 from half way, and one that is half way has at most 10 bits, which
// the step returns exactly (the residual of a representable quotient is exact in the fused operation).
//
// Both are one pass over memory: what bounds them is HBM beyond a few hundred tokens and the launch below.
#include "bw_cache.h"

namespace {

struct CacheArgs {
    const uint16_t *k, *v;
    int64_t k_row, k_head, v_row, v_head;
    const int64_t* slots;
    uint8_t *keys, *values;                      // cache
    uint32_t *key_meta, *value_meta;
    uint16_t *k_out, *v_out;
    int64_t rows;                                // pages * page_size
    int T, units, chunks, heads, groups, dim;    // units: threads of a token (2 * heads * chunks); chunks: dim / 8
    int page_shift, group_shift;                 // group / 8 = 1 << group_shift
};

// Row `row` of page `page` of a head: in rows, and in pairs of group g.
BW_DEV int64_t row_index(const CacheArgs& a, int64_t slot, int head) {
    const int64_t page = slot >> a.page_shift, row = slot & ((1 << a.page_shift) - 1);
    return ((page * a.heads + head) << a.page_shift) + row;
}
BW_DEV int64_t pair_index(const CacheArgs& a, int64_t slot, int head, int g) {
    const int64_t page = slot >> a.page_shift, row = slot & ((1 << a.page_shift) - 1);
    return (((page * a.heads + head) * a.groups + g) << a.page_shift) + row;
}

struct Unit { int token, head, chunk; bool value; };
BW_DEV Unit unit_of(const CacheArgs& a, uint32_t i) {
    Unit u;
    u.token = (int)(i / (uint32_t)a.units);
    uint32_t at = i - (uint32_t)u.token * a.units;
    u.value = at >= (uint32_t)a.units / 2;
    if (u.value) at -= a.units / 2;
    u.head = (int)(at / (uint32_t)a.chunks);
    u.chunk = (int)(at - (uint32_t)u.head * a.chunks);
    return u;
}

template <int DT, int BITS>
__global__ __launch_bounds__(256) void cache_write_kernel(CacheArgs a) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    const bool live = i < (uint32_t)a.T * (uint32_t)a.units;
    const Unit u = unit_of(a, live ? i : 0);
    const int64_t slot = a.slots[u.token];
    const bool kept = live && slot >= 0 && slot < a.rows;
    const uint16_t* src = u.value ? a.v + u.token * a.v_row + u.head * a.v_head : a.k + u.token * a.k_row + u.head * a.k_head;
    const u4 w = *reinterpret_cast<const u4*>(src + u.chunk * 8);
    uint8_t* out = u.value ? a.values : a.keys;
    if constexpr (BITS == 16) {
        if (kept) *reinterpret_cast<u4*>(out + (row_index(a, slot, u.head) * a.dim + u.chunk * 8) * 2) = w;
    } else {
        constexpr float top = (float)((1 << BITS) - 1);
        float x[8];
        float lo = 0.f, hi = 0.f, bad = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] = widen16<DT>((uint16_t)(w[j / 2] >> (16 * (j & 1))));
            lo = fminf(lo, x[j]);
            hi = fmaxf(hi, x[j]);
            bad = fmaxf(bad, __builtin_fabsf(x[j]) <= 3.402823466e38f ? 0.f : 1.f);
        }
        for (int o = 1; o < 1 << a.group_shift; o <<= 1) {
            lo = fminf(lo, __shfl_xor(lo, o, 64));
            hi = fmaxf(hi, __shfl_xor(hi, o, 64));
            bad = fmaxf(bad, __shfl_xor(bad, o, 64));
        }
        // the scale rounds up, so that no code has to be clipped for its rounding; never 0
        const float step = fminf(__fdiv_rn(__fsub_rn(hi, lo), top), 65504.f);
        uint16_t sb = __builtin_bit_cast(uint16_t, (_Float16)step);
        if ((float)__builtin_bit_cast(_Float16, sb) < step) sb++;
        if (sb == 0) sb = 1;
        const float s = (float)__builtin_bit_cast(_Float16, sb), r = __fdiv_rn(1.f, s);
        auto whole = [&](float v) {
            const float t = v * r;
            return rintf(__builtin_fmaf(__builtin_fmaf(-t, s, v), r, t));
        };
        const float z = fminf(whole(-lo), top);
        uint32_t words[BITS / 4] = {};
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float q = fminf(fmaxf(whole(x[j]) + z, 0.f), top);        // (a NaN: 0)
            words[j * BITS / 32] |= (uint32_t)q << (j * BITS % 32);
        }
        if (bad > 0.f) sb = 0x7E00;
        if (kept) {
            uint8_t* dst = out + row_index(a, slot, u.head) * (a.dim * BITS / 8) + u.chunk * BITS;
            if constexpr (BITS == 8) *reinterpret_cast<u2*>(dst) = u2{words[0], words[1]};
            else *reinterpret_cast<uint32_t*>(dst) = words[0];
            if ((u.chunk & ((1 << a.group_shift) - 1)) == 0)
                (u.value ? a.value_meta : a.key_meta)[pair_index(a, slot, u.head, u.chunk >> a.group_shift)] =
                    sb | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)z) << 16;
        }
    }
}

template <int DT, int BITS>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheArgs a) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint32_t)a.T * (uint32_t)a.units) return;
    const Unit u = unit_of(a, i);
    const int64_t slot = a.slots[u.token];
    const uint8_t* in = u.value ? a.values : a.keys;
    u4 w = {0, 0, 0, 0};
    if (slot >= 0 && slot < a.rows) {
        if constexpr (BITS == 16) {
            w = *reinterpret_cast<const u4*>(in + (row_index(a, slot, u.head) * a.dim + u.chunk * 8) * 2);
        } else {
            const uint8_t* src = in + row_index(a, slot, u.head) * (a.dim * BITS / 8) + u.chunk * BITS;
            const uint32_t pair = (u.value ? a.value_meta : a.key_meta)[pair_index(a, slot, u.head, u.chunk >> a.group_shift)];
            const float s = f16_bits(pair), z = f16_bits(pair >> 16);
            uint32_t words[BITS / 4];
            if constexpr (BITS == 8) { const u2 t = *reinterpret_cast<const u2*>(src); words[0] = t[0]; words[1] = t[1]; }
            else words[0] = *reinterpret_cast<const uint32_t*>(src);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float q = (float)((words[j * BITS / 32] >> (j * BITS % 32)) & ((1u << BITS) - 1));
                float x = s * (q - z);                                       // exact in float32: 11 bits times 9
                if (DT == BW_F16 && __builtin_fabsf(x) > 65504.f) x = __builtin_copysignf(65504.f, x);
                w[j / 2] |= (uint32_t)narrow16<DT>(x) << (16 * (j & 1));
            }
        }
    }
    uint16_t* out = (u.value ? a.v_out : a.k_out) + ((int64_t)u.token * a.heads + u.head) * a.dim + u.chunk * 8;
    *reinterpret_cast<u4*>(out) = w;
}

CacheArgs args_of(const bw_cache* c) {
    CacheArgs a = {};
    a.keys = (uint8_t*)c->keys;
    a.values = (uint8_t*)c->values;
    a.key_meta = (uint32_t*)c->key_meta;
    a.value_meta = (uint32_t*)c->value_meta;
    a.rows = c->pages * c->page_size;
    a.heads = c->kv_heads;
    a.dim = c->dim;
    a.chunks = c->dim / 8;
    a.units = 2 * c->kv_heads * a.chunks;
    a.page_shift = bw_log2(c->page_size);
    if (c->bits != 16) {
        a.groups = c->dim / c->group;
        a.group_shift = bw_log2(c->group / 8);
    }
    return a;
}

// Runs `launch(args, blocks)` over the tokens, in several launches where a thread's number would pass 31 bits.
template <class F>
int over_tokens(CacheArgs a, int64_t T, F&& launch) {
    const int64_t most = ((int64_t)1 << 31) / a.units - 1;
    for (int64_t at = 0; at < T; at += most) {
        CacheArgs b = a;
        b.T = (int)(T - at < most ? T - at : most);
        b.slots += at;
        if (b.k) { b.k += at * a.k_row; b.v += at * a.v_row; }
        if (b.k_out) { b.k_out += at * a.heads * a.dim; b.v_out += at * a.heads * a.dim; }
        launch(b, dim3((unsigned)(((int64_t)b.T * a.units + 255) / 256)));
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    return BW_OK;
}

}  // namespace

#define BW_BY_FORMAT(KERNEL, DT)                                                                                          \
    over_tokens(a, T, [&](const CacheArgs& b, dim3 grid) {                                                                \
        if (c->bits == 16) hipLaunchKernelGGL((KERNEL<DT, 16>), grid, dim3(256), 0, (hipStream_t)stream, b);              \
        else if (c->bits == 8) hipLaunchKernelGGL((KERNEL<DT, 8>), grid, dim3(256), 0, (hipStream_t)stream, b);           \
        else hipLaunchKernelGGL((KERNEL<DT, 4>), grid, dim3(256), 0, (hipStream_t)stream, b);                             \
    })

extern "C" int bw_cache_write(const bw_cache* c, int act_dtype, int64_t T, const void* k, int64_t k_row, int64_t k_head, const void* v,
                              int64_t v_row, int64_t v_head, const int64_t* slots, void* stream) {
    if (int st = bw_cache_check(c)) return st;
    if (T < 0 || (T > 0 && (!k || !v || !slots))) return BW_EINVAL;
    if ((act_dtype != BW_F16 && act_dtype != BW_BF16) || (c->bits == 16 && act_dtype != c->dtype)) return BW_EUNSUPPORTED;
    if (T == 0) return BW_OK;
    if (!bw_aligned(k, 16) || !bw_aligned(v, 16) || !bw_aligned(slots, 8) || (k_row | k_head | v_row | v_head) % 8) return BW_EALIGN;
    CacheArgs a = args_of(c);
    a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
    a.k_row = k_row; a.k_head = k_head; a.v_row = v_row; a.v_head = v_head;
    a.slots = slots;
    return act_dtype == BW_F16 ? BW_BY_FORMAT(cache_write_kernel, BW_F16) : BW_BY_FORMAT(cache_write_kernel, BW_BF16);
}

extern "C" int bw_cache_read(const bw_cache* c, int out_dtype, int64_t T, const int64_t* slots, void* k_out, void* v_out, void* stream) {
    if (int st = bw_cache_check(c)) return st;
    if (T < 0 || (T > 0 && (!slots || !k_out || !v_out))) return BW_EINVAL;
    if ((out_dtype != BW_F16 && out_dtype != BW_BF16) || (c->bits == 16 && out_dtype != c->dtype)) return BW_EUNSUPPORTED;
    if (T == 0) return BW_OK;
    if (!bw_aligned(k_out, 16) || !bw_aligned(v_out, 16) || !bw_aligned(slots, 8)) return BW_EALIGN;
    CacheArgs a = args_of(c);
    a.slots = slots;
    a.k_out = (uint16_t*)k_out; a.v_out = (uint16_t*)v_out;
    return out_dtype == BW_F16 ? BW_BY_FORMAT(cache_read_kernel, BW_F16) : BW_BY_FORMAT(cache_read_kernel, BW_BF16);
}
