// Attention of one new token of each sequence over its paged key-value cache: the C entry point, the join of sequences that lie in several
// pieces, and the 16-bit instantiations of the kernel in bw_attention_kernel.h (bw_attention_w8.hip and bw_attention_w4.hip hold the others).
#include "bw_attention_kernel.h"

#include "bw_attention.h"

namespace {

// One workgroup for 128 values of the output [queries][dim] of the segment that piece blockIdx.x / chunks began and left unfinished, if it did: 32
// threads of 4 values each, ROWS such rows that share the parts, four parts of a thread under way at a time.  What bounds it is the way to
// memory and back twice (the joint, the parts) and the number of threads that are launched to find nothing: two rows unless segments are so few that
// each has 8 pieces and more (16 sequences of 1024, 8 heads of 128: 24.0 us with two, 24.8 with 8, 27 with 16; one sequence of 65537: 31.6, 26.6, 26.2).
constexpr int kJoinValues = 128, kJoinAhead = 4, kManyParts = 8;
template <int ROWS>
__global__ __launch_bounds__(32 * ROWS) void attention_join_kernel(AttentionArgs a, int chunks) {
    __shared__ float tops[ROWS][32], sums[ROWS][32];
    __shared__ f4 outs[ROWS][32];
    const uint32_t w0 = blockIdx.x / (uint32_t)chunks, chunk = blockIdx.x - w0 * chunks;
    const Joint joint = a.joints[w0];
    if (joint.parts == 0) return;
    const uint32_t b = joint.b, hq = joint.hq, w1 = w0 + joint.parts - 1;
    const int head = (int)(hq / (uint32_t)a.q_groups), first_query = (int)(hq - (uint32_t)head * a.q_groups) * kQueries;
    const int queries = a.share - first_query < kQueries ? a.share - first_query : kQueries;
    const int x = (int)threadIdx.x & 31, y = (int)threadIdx.x >> 5;
    const int e = ((int)chunk * 32 + x) * 4, query = e / a.dim;
    const bool live = query < queries;
    const int64_t pitch = 2 * kQueries + a.queries * a.dim;
    float top = -INFINITY, sum = 0.f;
    f4 o = {0.f, 0.f, 0.f, 0.f};
    if (live) {
        for (uint32_t w = w0 + y; w <= w1; w += kJoinAhead * ROWS) {
            float r[kJoinAhead], l[kJoinAhead];
            f4 v[kJoinAhead];
#pragma unroll
            for (int i = 0; i < kJoinAhead; i++) {
                const uint32_t part = w + i * ROWS;
                const float* p = a.partial + (2 * (int64_t)(part <= w1 ? part : w) + (part == w0)) * pitch;
                r[i] = part <= w1 ? p[query] : -INFINITY;
                l[i] = p[kQueries + query];
                v[i] = *reinterpret_cast<const f4*>(p + 2 * kQueries + e);
            }
            float now = top;
#pragma unroll
            for (int i = 0; i < kJoinAhead; i++) now = fmaxf(now, r[i]);
            const float keep = top == now ? 1.f : __builtin_amdgcn_exp2f(top - now);
            top = now;
            sum *= keep;
            o *= keep;
#pragma unroll
            for (int i = 0; i < kJoinAhead; i++) {
                if (w + i * ROWS > w1) break;
                const float f = r[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(r[i] - top);
                sum += f * l[i];
                o += f * v[i];
            }
        }
    }
    tops[y][x] = top;
    sums[y][x] = sum;
    outs[y][x] = o;
    __syncthreads();
    if (y || !live) return;
#pragma unroll
    for (int i = 1; i < ROWS; i++) top = fmaxf(top, tops[i][x]);
    o = f4{0.f, 0.f, 0.f, 0.f};
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const float f = tops[i][x] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(tops[i][x] - top);
        sum += f * sums[i][x];
        o += f * outs[i][x];
    }
    const float inv = top == -INFINITY ? 0.f : 1.f / sum;           // no tokens: 0; none with a finite score: 0 / 0
    store_out(a, (int64_t)b * a.q_heads + head * a.share + first_query + query, e - query * a.dim, o * inv);
}

int attention_check(const bw_cache* c, int64_t B, int q_heads, int64_t max_pages) {
    if (int st = bw_cache_check(c)) return st;
    if (B < 0 || q_heads < 1 || q_heads % c->kv_heads || max_pages < 1) return BW_EINVAL;
    if (B > 1 << 20 || q_heads > 65535 || max_pages >= ((int64_t)1 << 25) / c->page_size) return BW_EUNSUPPORTED;
    if (B * ((max_pages * c->page_size + kTile - 1) / kTile + kSegmentCost) >= ((int64_t)1 << 31) / q_heads || B * q_heads >= (int64_t)1 << 29) return BW_EUNSUPPORTED;
    return BW_OK;
}

// Workgroups, and whether every segment gets one of its own: nothing to cut, nothing to join.  With room for 512 tokens to a sequence always (128
// sequences of 12 heads of 64: 15.3 us against 20.0), with room for 1024 where there are segments for half the CUs at least (64 sequences of up to
// 1000, 8 heads of 128 in 4 bits: 16.6 against 22.4; 4 such sequences: 15.2 against 10.1), beyond never (32 of up to 2000 in 8 bits: 28.7 against 22.0).
// (With a window there is room for its tiles and the sinks', however long the table.)
struct Plan { uint32_t grid; bool whole; };
constexpr int kWholeTokens = 512, kWholeMany = 1024;
struct Window { int64_t tokens, sinks; };                        // tokens 0: all
Plan plan_of(const bw_cache* c, int64_t B, int q_heads, int64_t max_pages, Window w) {
    const int64_t share = q_heads / c->kv_heads, segments = B * c->kv_heads * ((share + kQueries - 1) / kQueries), room = max_pages * c->page_size;
    const int64_t seen = w.tokens && w.tokens < room && w.sinks < room ? ((w.tokens + kTile - 1) / kTile + 1 + (w.sinks + kTile - 1) / kTile) * kTile : room, tokens = seen < room ? seen : room;
    const int cus = bw_device_cus();
    Plan p;
    p.whole = tokens <= (2 * segments >= cus ? kWholeMany : kWholeTokens) && segments < (int64_t)1 << 24;          // (2^32 threads of a launch)
    // (no more than there can be pieces: workgroups that find nothing cost their launch)
    const int64_t resident = (int64_t)cus * resident_workgroups(c->dim);
    const int64_t pieces = (segments * ((tokens + kTile - 1) / kTile + kSegmentCost) + kWaves - 1) / kWaves;
    p.grid = (uint32_t)(p.whole ? segments : resident < pieces ? resident : pieces);
    return p;
}

}  // namespace

static size_t workspace_bytes_of(const bw_cache* c, int64_t B, int q_heads, int64_t max_pages, Window w) {
    if (attention_check(c, B, q_heads, max_pages) != BW_OK || B == 0 || w.tokens < 0 || w.sinks < 0) return 0;
    const Plan p = plan_of(c, B, q_heads, max_pages, w);
    const int share = q_heads / c->kv_heads, queries = share < kQueries ? share : kQueries;
    return p.whole ? 0 : (size_t)p.grid * (sizeof(Joint) + 2 * (2 * kQueries + queries * c->dim) * sizeof(float));
}

static int attend(const bw_cache* c, int act_dtype, const void* q, int64_t B, int q_heads, int64_t q_row, int64_t q_head, const int32_t* page_table, int64_t max_pages,
                  int64_t table_row, const int32_t* lengths, float scale, Window w, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (int st = attention_check(c, B, q_heads, max_pages)) return st;
    if (w.tokens < 0 || w.sinks < 0) return BW_EINVAL;
    if ((act_dtype != BW_F16 && act_dtype != BW_BF16) || (c->bits == 16 && act_dtype != c->dtype)) return BW_EUNSUPPORTED;
    if (B == 0) return BW_OK;
    if (!q || !page_table || !lengths || !out) return BW_EINVAL;
    if (table_row < max_pages && B > 1 && table_row != 0) return BW_EINVAL;
    if (!bw_aligned(q, 16) || !bw_aligned(out, 16) || !bw_aligned(page_table, 4) || !bw_aligned(lengths, 4) || (q_row | q_head) % 8) return BW_EALIGN;
    const Plan plan = plan_of(c, B, q_heads, max_pages, w);
    const size_t bytes = workspace_bytes_of(c, B, q_heads, max_pages, w);
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
    a.joints = (Joint*)workspace;
    a.partial = (float*)(a.joints + plan.grid);
    a.pages = (uint32_t)c->pages;
    a.B = (int)B;
    a.q_heads = q_heads; a.kv_heads = c->kv_heads; a.share = q_heads / c->kv_heads;
    a.queries = a.share < kQueries ? a.share : kQueries;
    a.q_groups = (a.share + kQueries - 1) / kQueries;
    a.dim = c->dim; a.row_bytes = c->dim * c->bits / 8;
    a.page_shift = bw_log2(c->page_size);
    a.max_tokens = (int)(max_pages * c->page_size);
    a.window = w.tokens && w.tokens < a.max_tokens ? (int)w.tokens : a.max_tokens;
    a.sinks = w.sinks < a.max_tokens ? (int)w.sinks : a.max_tokens;
    a.q_bf16 = act_dtype == BW_BF16;
    a.cus = bw_device_cus();
    a.whole = plan.whole;
    a.scale = scale * 1.44269504088896340736f;
    const hipStream_t st = (hipStream_t)stream;
    if (c->bits == 8) bw_launch_attention_w8(a, c->group, plan.grid, st);
    else if (c->bits == 4) bw_launch_attention_w4(a, c->group, plan.grid, st);
    else if (c->dtype == BW_F16) {
        if (c->dim <= 64) launch_attention<Format16<BW_F16, 64>, 1>(a, plan.grid, st);
        else if (c->dim <= 128) launch_attention<Format16<BW_F16, 128>, 1>(a, plan.grid, st);
        else launch_attention<Format16<BW_F16, 256>, 1>(a, plan.grid, st);
    } else {
        if (c->dim <= 64) launch_attention<Format16<BW_BF16, 64>, 1>(a, plan.grid, st);
        else if (c->dim <= 128) launch_attention<Format16<BW_BF16, 128>, 1>(a, plan.grid, st);
        else launch_attention<Format16<BW_BF16, 256>, 1>(a, plan.grid, st);
    }
    if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    if (!plan.whole) {
        const int chunks = (a.queries * a.dim + kJoinValues - 1) / kJoinValues;
        if ((int64_t)plan.grid >= kManyParts * B * c->kv_heads * a.q_groups) hipLaunchKernelGGL(attention_join_kernel<8>, dim3(plan.grid * chunks), dim3(256), 0, st, a, chunks);
        else hipLaunchKernelGGL(attention_join_kernel<2>, dim3(plan.grid * chunks), dim3(64), 0, st, a, chunks);
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    return BW_OK;
}

extern "C" size_t bw_cache_attention_workspace_bytes(const bw_cache* c, int64_t B, int q_heads, int64_t max_pages) {
    return workspace_bytes_of(c, B, q_heads, max_pages, Window{0, 0});
}

extern "C" int bw_cache_attention(const bw_cache* c, int act_dtype, const void* q, int64_t B, int q_heads, int64_t q_row, int64_t q_head,
                                  const int32_t* page_table, int64_t max_pages, int64_t table_row, const int32_t* lengths, float scale, void* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    return attend(c, act_dtype, q, B, q_heads, q_row, q_head, page_table, max_pages, table_row, lengths, scale, Window{0, 0}, out, workspace, workspace_bytes, stream);
}

extern "C" size_t bw_cache_attention_window_workspace_bytes(const bw_cache* c, int64_t B, int q_heads, int64_t max_pages, int64_t window, int64_t sinks) {
    return workspace_bytes_of(c, B, q_heads, max_pages, Window{window, sinks});
}

extern "C" int bw_cache_attention_window(const bw_cache* c, int act_dtype, const void* q, int64_t B, int q_heads, int64_t q_row, int64_t q_head,
                                         const int32_t* page_table, int64_t max_pages, int64_t table_row, const int32_t* lengths, float scale, int64_t window,
                                         int64_t sinks, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    return attend(c, act_dtype, q, B, q_heads, q_row, q_head, page_table, max_pages, table_row, lengths, scale, Window{window, sinks}, out, workspace, workspace_bytes, stream);
}
