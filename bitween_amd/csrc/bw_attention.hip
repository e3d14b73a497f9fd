// Attention of one new token of each sequence over its paged key-value cache.
//
// One workgroup for each sequence and query head; its waves take the cached tokens in turn, each with a running maximum and sum, and are
// joined through LDS.  A lane holds the values of a head at lane, lane + 64, ...
#include "bw_cache.h"

namespace {

struct AttentionArgs {
    const uint16_t* q;
    int64_t q_row, q_head;
    const int32_t *table, *lengths;
    int64_t table_row;
    const uint8_t *keys, *values;
    const uint32_t *key_meta, *value_meta;
    uint16_t* out;
    int64_t pages;
    int q_heads, kv_heads, share, dim, bits, group, groups, page_shift, max_pages, q_bf16, cache_bf16;
    float scale;
};

BW_DEV float cached(const AttentionArgs& a, const uint8_t* base, const uint32_t* meta, int64_t page, int head, int row, int d) {
    const int64_t at = ((page * a.kv_heads + head) << a.page_shift) + row;
    if (a.bits == 16) {
        const uint16_t u = ((const uint16_t*)base)[at * a.dim + d];
        return a.cache_bf16 ? bf16_to_f32(u) : f16_bits(u);
    }
    const uint32_t w = ((const uint32_t*)base)[at * (a.dim * a.bits / 32) + d * a.bits / 32];
    const uint32_t pair = meta[(((page * a.kv_heads + head) * a.groups + d / a.group) << a.page_shift) + row];
    return f16_bits(pair) * ((float)((w >> (d * a.bits % 32)) & ((1u << a.bits) - 1)) - f16_bits(pair >> 16));
}

__global__ __launch_bounds__(256) void attention_kernel(AttentionArgs a) {
    __shared__ float part[4][256];
    __shared__ float stat[4][2];
    const int b = (int)blockIdx.x / a.q_heads, h = (int)blockIdx.x - b * a.q_heads, head = h / a.share;
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    int64_t n = a.lengths[b];
    const int64_t room = (int64_t)a.max_pages << a.page_shift;
    if (n > room) n = room;
    float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = lane + 64 * i;
        const uint16_t u = d < a.dim ? a.q[b * a.q_row + h * a.q_head + d] : 0;
        q[i] = (a.q_bf16 ? bf16_to_f32(u) : f16_bits(u)) * a.scale;
    }
    for (int64_t t = wave; t < n; t += 4) {
        const int64_t page = a.table[b * a.table_row + (t >> a.page_shift)];
        if (page < 0 || page >= a.pages) continue;
        const int row = (int)(t & ((1 << a.page_shift) - 1));
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < a.dim) s += q[i] * cached(a, a.keys, a.key_meta, page, head, row, lane + 64 * i);
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        const float top = fmaxf(m, s);
        const float keep = m == top ? 1.f : __expf(m - top), p = __expf(s - top);
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 64 * i < a.dim) acc[i] = acc[i] * keep + p * cached(a, a.values, a.value_meta, page, head, row, lane + 64 * i);
        m = top;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) part[wave][lane + 64 * i] = acc[i];
    if (lane == 0) { stat[wave][0] = m; stat[wave][1] = l; }
    __syncthreads();
    const int d = (int)threadIdx.x;
    if (d >= a.dim) return;
    const float top = fmaxf(fmaxf(stat[0][0], stat[1][0]), fmaxf(stat[2][0], stat[3][0]));
    float num = 0.f, den = 0.f;
    for (int w = 0; w < 4; w++) {
        if (stat[w][1] == 0.f) continue;
        const float f = __expf(stat[w][0] - top);
        num += f * part[w][d];
        den += f * stat[w][1];
    }
    const float o = den == 0.f ? 0.f : num / den;
    a.out[((int64_t)b * a.q_heads + h) * a.dim + d] = a.q_bf16 ? f32_to_bf16(o) : __builtin_bit_cast(uint16_t, (_Float16)o);
}

int attention_check(const bw_cache* c, int64_t B, int q_heads, int64_t max_pages) {
    if (int st = bw_cache_check(c)) return st;
    if (B < 0 || q_heads < 1 || q_heads % c->kv_heads || max_pages < 1) return BW_EINVAL;
    if (B > 1 << 20 || q_heads > 65535 || B * q_heads >= (int64_t)1 << 31 || max_pages * c->page_size >= (int64_t)1 << 31) return BW_EUNSUPPORTED;
    return BW_OK;
}

}  // namespace

extern "C" size_t bw_cache_attention_workspace_bytes(const bw_cache* c, int64_t B, int q_heads, int64_t max_pages) { return 0; }

extern "C" int bw_cache_attention(const bw_cache* c, int act_dtype, const void* q, int64_t B, int q_heads, int64_t q_row, int64_t q_head,
                                  const int32_t* page_table, int64_t max_pages, int64_t table_row, const int32_t* lengths, float scale, void* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    if (int st = attention_check(c, B, q_heads, max_pages)) return st;
    if ((act_dtype != BW_F16 && act_dtype != BW_BF16) || (c->bits == 16 && act_dtype != c->dtype)) return BW_EUNSUPPORTED;
    if (B == 0) return BW_OK;
    if (!q || !page_table || !lengths || !out) return BW_EINVAL;
    if (table_row < max_pages && B > 1 && table_row != 0) return BW_EINVAL;
    if (!bw_aligned(q, 16) || !bw_aligned(out, 16) || !bw_aligned(page_table, 4) || !bw_aligned(lengths, 4) || (q_row | q_head) % 8) return BW_EALIGN;
    AttentionArgs a = {};
    a.q = (const uint16_t*)q; a.q_row = q_row; a.q_head = q_head;
    a.table = page_table; a.lengths = lengths; a.table_row = table_row;
    a.keys = (const uint8_t*)c->keys; a.values = (const uint8_t*)c->values;
    a.key_meta = (const uint32_t*)c->key_meta; a.value_meta = (const uint32_t*)c->value_meta;
    a.out = (uint16_t*)out;
    a.pages = c->pages;
    a.q_heads = q_heads; a.kv_heads = c->kv_heads; a.share = q_heads / c->kv_heads;
    a.dim = c->dim; a.bits = c->bits; a.group = c->bits == 16 ? c->dim : c->group; a.groups = c->dim / a.group;
    a.page_shift = bw_log2(c->page_size); a.max_pages = (int)max_pages;
    a.q_bf16 = act_dtype == BW_BF16; a.cache_bf16 = c->dtype == BW_BF16;
    a.scale = scale;
    hipLaunchKernelGGL(attention_kernel, dim3((unsigned)(B * q_heads)), dim3(256), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? BW_OK : BW_ELAUNCH;
}
