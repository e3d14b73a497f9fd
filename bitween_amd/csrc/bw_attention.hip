// Attention of one new token of each sequence over its paged key-value cache: the C entry point, the join of sequences that lie in several
// pieces, and the 16-bit instantiations of the kernel in bw_attention_kernel.h (bw_attention_w8.hip and bw_attention_w4.hip hold the others).
#include "bw_attention_kernel.h"

#include "bw_attention.h"

namespace {

// One workgroup for 128 values of a segment's output [queries][dim]: 32 threads of 4 values each, eight such rows that share the pieces.
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a, uint32_t grid, int chunks) {
    __shared__ uint32_t lds[8];
    __shared__ float tops[8][32];
    __shared__ f4 outs[8][32];
    __shared__ float sums[8][32];
    const uint32_t segment = blockIdx.x / (uint32_t)chunks, chunk = blockIdx.x - segment * chunks, per_seq = (uint32_t)(a.kv_heads * a.q_groups);
    const uint32_t b = segment / per_seq, hq = segment - b * per_seq;
    uint32_t all;
    scan_sequences(a, lds, all, [&](uint32_t, uint32_t, uint32_t) { return true; },
                   [&](int b_, uint32_t before) { if ((uint32_t)b_ == b) lds[4] = before; });
    const uint32_t tiles = tiles_of(tokens_of(a, (int)b));
    if (tiles == 0) return;
    const Split s = split_of(a, all, grid);
    const uint64_t first = (uint64_t)lds[4] * per_seq + (uint64_t)hq * tiles;
    const uint32_t w0 = s.piece_of(first), w1 = s.piece_of(first + tiles - 1);
    if (w0 == w1) return;
    const int head = (int)(hq / (uint32_t)a.q_groups), first_query = (int)(hq - (uint32_t)head * a.q_groups) * kQueries;
    const int queries = a.share - first_query < kQueries ? a.share - first_query : kQueries;
    const int x = (int)threadIdx.x & 31, y = (int)threadIdx.x >> 5;
    const int e = ((int)chunk * 32 + x) * 4, query = e / a.dim;
    const bool live = query < queries;
    const int64_t pitch = 2 * kQueries + a.queries * a.dim;
    auto slot = [&](uint32_t w) { return a.partial + (2 * (int64_t)w + (w == w0)) * pitch; };
    float top = -INFINITY;
    if (live)
        for (uint32_t w = w0 + y; w <= w1; w += 8) top = fmaxf(top, slot(w)[query]);
    tops[y][x] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) top = fmaxf(top, tops[i][x]);
    f4 o = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
    if (live)
        for (uint32_t w = w0 + y; w <= w1; w += 8) {
            const float* p = slot(w);
            const float r = p[query], f = r == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r - top);
            sum += f * p[kQueries + query];
            o += f * *reinterpret_cast<const f4*>(p + 2 * kQueries + e);
        }
    outs[y][x] = o;
    sums[y][x] = sum;
    __syncthreads();
    if (y || !live) return;
#pragma unroll
    for (int i = 1; i < 8; i++) {
        o += outs[i][x];
        sum += sums[i][x];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    store_out(a, (int64_t)b * a.q_heads + head * a.share + first_query + query, e - query * a.dim, o * inv);
}

int attention_check(const bw_cache* c, int64_t B, int q_heads, int64_t max_pages) {
    if (int st = bw_cache_check(c)) return st;
    if (B < 0 || q_heads < 1 || q_heads % c->kv_heads || max_pages < 1) return BW_EINVAL;
    if (B > 1 << 20 || q_heads > 65535 || B * q_heads >= (int64_t)1 << 31 || max_pages * c->page_size >= (int64_t)1 << 25) return BW_EUNSUPPORTED;
    if (B * ((max_pages * c->page_size + kTile - 1) / kTile) >= (int64_t)1 << 31 || B * q_heads * ((c->dim + 127) / 128 + 1) >= (int64_t)1 << 31) return BW_EUNSUPPORTED;
    return BW_OK;
}

// Workgroups, and whether every segment gets one of its own.
struct Plan { uint32_t grid; bool whole; };
constexpr int kMinTiles = 8, kWholeTokens = 512;
Plan plan_of(const bw_cache* c, int64_t B, int q_heads, int64_t max_pages) {
    const int64_t share = q_heads / c->kv_heads, segments = B * c->kv_heads * ((share + kQueries - 1) / kQueries);
    Plan p;
    p.whole = max_pages * c->page_size <= kWholeTokens && segments < (int64_t)1 << 31;
    p.grid = p.whole ? (uint32_t)segments : (uint32_t)bw_device_cus() * 2;
    return p;
}

}  // namespace

template <class F> static void launch(const AttentionArgs& a, uint32_t grid, hipStream_t stream) {
    hipLaunchKernelGGL(attention_kernel<F>, dim3(grid), dim3(256), 0, stream, a);
}

extern "C" size_t bw_cache_attention_workspace_bytes(const bw_cache* c, int64_t B, int q_heads, int64_t max_pages) {
    if (attention_check(c, B, q_heads, max_pages) != BW_OK || B == 0) return 0;
    const Plan p = plan_of(c, B, q_heads, max_pages);
    const int share = q_heads / c->kv_heads, queries = share < kQueries ? share : kQueries;
    return p.whole ? 0 : (size_t)p.grid * 2 * (2 * kQueries + queries * c->dim) * sizeof(float);
}

extern "C" int bw_cache_attention(const bw_cache* c, int act_dtype, const void* q, int64_t B, int q_heads, int64_t q_row, int64_t q_head,
                                  const int32_t* page_table, int64_t max_pages, int64_t table_row, const int32_t* lengths, float scale, void* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    if (int st = attention_check(c, B, q_heads, max_pages)) return st;
    if ((act_dtype != BW_F16 && act_dtype != BW_BF16) || (c->bits == 16 && act_dtype != c->dtype)) return BW_EUNSUPPORTED;
    if (B == 0) return BW_OK;
    if (!q || !page_table || !lengths || !out) return BW_EINVAL;
    if (table_row < max_pages && B > 1 && table_row != 0) return BW_EINVAL;
    if (!bw_aligned(q, 16) || !bw_aligned(out, 16) || !bw_aligned(page_table, 4) || !bw_aligned(lengths, 4) || (q_row | q_head) % 8) return BW_EALIGN;
    const Plan plan = plan_of(c, B, q_heads, max_pages);
    const size_t bytes = bw_cache_attention_workspace_bytes(c, B, q_heads, max_pages);
    if (bytes) {
        if (!workspace || workspace_bytes < bytes) return BW_EWORKSPACE;
        if (!bw_aligned(workspace, 16)) return BW_EALIGN;
    }
    AttentionArgs a = {};
    a.q = (const uint16_t*)q; a.q_row = q_row; a.q_head = q_head;
    a.table = page_table; a.lengths = lengths; a.table_row = table_row;
    a.keys = (const uint8_t*)c->keys; a.values = (const uint8_t*)c->values;
    a.key_meta = (const uint32_t*)c->key_meta; a.value_meta = (const uint32_t*)c->value_meta;
    a.out = (uint16_t*)out;
    a.partial = (float*)workspace;
    a.pages = (uint32_t)c->pages;
    a.B = (int)B;
    a.q_heads = q_heads; a.kv_heads = c->kv_heads; a.share = q_heads / c->kv_heads;
    a.queries = a.share < kQueries ? a.share : kQueries;
    a.q_groups = (a.share + kQueries - 1) / kQueries;
    a.dim = c->dim; a.row_bytes = c->dim * c->bits / 8;
    a.page_shift = bw_log2(c->page_size);
    a.max_tokens = (int)(max_pages * c->page_size);
    a.q_bf16 = act_dtype == BW_BF16;
    a.min_tiles = kMinTiles;
    a.whole = plan.whole;
    a.scale = scale * 1.44269504088896340736f;
    const hipStream_t st = (hipStream_t)stream;
    if (c->bits == 8) bw_launch_attention_w8(a, c->group, plan.grid, st);
    else if (c->bits == 4) bw_launch_attention_w4(a, c->group, plan.grid, st);
    else if (c->dtype == BW_F16) {
        if (c->dim <= 64) launch<Format16<BW_F16, 64>>(a, plan.grid, st);
        else if (c->dim <= 128) launch<Format16<BW_F16, 128>>(a, plan.grid, st);
        else launch<Format16<BW_F16, 256>>(a, plan.grid, st);
    } else {
        if (c->dim <= 64) launch<Format16<BW_BF16, 64>>(a, plan.grid, st);
        else if (c->dim <= 128) launch<Format16<BW_BF16, 128>>(a, plan.grid, st);
        else launch<Format16<BW_BF16, 256>>(a, plan.grid, st);
    }
    if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    if (!plan.whole) {
        const int chunks = (a.queries * a.dim + 127) / 128;
        hipLaunchKernelGGL(attention_join_kernel, dim3((unsigned)(B * a.kv_heads * a.q_groups * chunks)), dim3(256), 0, st, a, plan.grid, chunks);
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    return BW_OK;
}
