// Causal attention of many tokens of each sequence (prompts, training), with a window and sinks, and its gradients: the C entry points, and the joins of what was
// cut into parts.  The kernels are in bw_prompt_kernel.h and bw_prompt_grad_kernel.h, instantiated by bw_prompt_*.hip for each type.
#include "bw_prompt_grad.h"

#include <utility>

namespace {

// out = the parts of a row put together: [row][part] reference and sum, then [row][part][dim] sums of the values.  A thread has 4 values of a row, and 8 parts under way at a
// time (one at a time: 28.6 us for 2016 rows of 128 in 32 parts).
template <int DT>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs a, int threads, uint32_t rows) {
    const uint32_t i = blockIdx.x * (256 / threads) + threadIdx.x / threads;
    const int d = (int)(threadIdx.x % threads) * 4;
    if (threadIdx.x / threads >= 256 / threads || i >= rows) return;
    const u2* stats = reinterpret_cast<const u2*>(a.partial) + (int64_t)i * a.splits;
    const float* part = a.partial + (int64_t)rows * a.splits * 2 + (int64_t)i * a.splits * a.dim + d;
    float top = -INFINITY, sum = 0.f;
    f4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; s += 8) {
        f4 x[8];
        float r[8], l[8], high = top;
#pragma unroll
        for (int n = 0; n < 8; n++) {
            const int at = s + n < a.splits ? s + n : s;
            const u2 w = stats[at];
            const uint32_t first = w[0], second = w[1];
            r[n] = s + n < a.splits ? __builtin_bit_cast(float, first) : -INFINITY;
            l[n] = __builtin_bit_cast(float, second);
            x[n] = *reinterpret_cast<const f4*>(part + (int64_t)at * a.dim);
            high = fmaxf(high, r[n]);
        }
        if (high == -INFINITY) continue;                           // no key of these parts is seen
        const float keep = __builtin_amdgcn_exp2f(top - high);
        top = high;
        sum *= keep;
        o *= keep;
#pragma unroll
        for (int n = 0; n < 8; n++) {
            if (r[n] == -INFINITY) continue;                       // (nothing was summed)
            const float f = __builtin_amdgcn_exp2f(r[n] - top);
            sum += f * l[n];
            o += f * x[n];
        }
    }
    const bool empty = top == -INFINITY;
    o *= empty ? 0.f : 1.f / sum;
    uint32_t rest;
    const uint32_t token_head = i / (uint32_t)a.share, j = i - token_head * a.share, head = token_head / (uint32_t)a.q_tokens;
    rest = token_head - head * a.q_tokens;
    store4<DT>(a.out + ((int64_t)rest * a.q_heads + head * a.share + j) * a.dim + d, o[0], o[1], o[2], o[3]);
    if (a.lse && d == 0) a.lse[i] = empty ? INFINITY : top + __builtin_amdgcn_logf(sum);
}

int prompt_check(const bw_prompt* p, int act_dtype) {
    if (!p || p->q_tokens < 0 || p->k_tokens < 0 || p->sequences < 1 || p->q_heads < 1 || p->kv_heads < 1 || p->q_heads % p->kv_heads || p->dim < 1 || p->window < 0 ||
        p->sinks < 0)
        return BW_EINVAL;
    if (!p->q_starts != !p->k_starts) return BW_EINVAL;
    if (!p->q_starts && (p->q_tokens % p->sequences || p->k_tokens % p->sequences)) return BW_EINVAL;
    if (act_dtype != BW_F16 && act_dtype != BW_BF16) return BW_EUNSUPPORTED;
    if (p->dim % 8 || p->dim > 256 || p->q_heads > 65535 || p->sequences > 1 << 20) return BW_EUNSUPPORTED;
    if (p->q_tokens >= (int64_t)1 << 31 || p->k_tokens >= (int64_t)1 << 31 || p->q_tokens + p->k_tokens >= ((int64_t)1 << 31) - 1024) return BW_EUNSUPPORTED;
    if (p->q_tokens * p->q_heads >= (int64_t)1 << 31 || (p->k_tokens + p->q_tokens) * p->kv_heads >= (int64_t)1 << 31) return BW_EUNSUPPORTED;
    if (!bw_aligned(p->q_starts, 4) || !bw_aligned(p->k_starts, 4)) return BW_EALIGN;
    return BW_OK;
}

// Workgroups of `tile` rows (or keys) each: of a sequence, or slots for all of them.
int64_t tiles_of(const bw_prompt* p, int64_t tokens, int share, int tile) {
    return p->q_starts ? tokens * share / tile + p->sequences + 2 : (tokens / p->sequences * share + tile - 1) / tile;
}

PromptArgs args_of(const bw_prompt* p) {
    PromptArgs a = {};
    a.q_starts = p->q_starts; a.k_starts = p->k_starts;
    a.q_tokens = (int)p->q_tokens; a.k_tokens = (int)p->k_tokens;
    a.sequences = p->sequences;
    a.seq_q = (int)(p->q_tokens / p->sequences); a.seq_k = (int)(p->k_tokens / p->sequences);
    a.q_heads = p->q_heads; a.kv_heads = p->kv_heads; a.share = p->q_heads / p->kv_heads;
    a.dim = p->dim;
    // (a window of all tokens hides none)
    a.window = (int)(p->window && p->window < p->k_tokens ? p->window : p->k_tokens > 0 ? p->k_tokens : 1);
    a.sinks = (int)(p->sinks < p->k_tokens ? p->sinks : p->k_tokens);
    a.combos = (uint32_t)(p->kv_heads * (int64_t)(p->q_starts ? 1 : p->sequences));
    a.by_share = FastDiv((uint32_t)a.share);
    a.by_combos = FastDiv(a.combos);
    a.by_heads = FastDiv((uint32_t)p->kv_heads);
    a.flip = p->scale < 0.f ? 0x80008000u : 0u;
    // (scale 0: all scores that are numbers weigh the same, and hidden ones, minus infinity, stay hidden: the smallest number, which makes 2^-21 of the largest score)
    const float scale = __builtin_fabsf(p->scale) * 1.44269504088896340736f;
    a.scale = scale == 0.f ? __FLT_DENORM_MIN__ : scale;
    return a;
}

int key_tile(int dim) { return dim > 128 ? 32 : 64; }

// Parts that the keys of a tile of rows are cut into, and waves' groups of a workgroup (see prompt_forward_kernel): what takes the least by this count, in microseconds, as measured.
// A tile of keys takes a workgroup 0.9 (heads of 64), 1.36 (96), 1.5 (128) or 1.7 (256, of half the keys); where two share a CU, each a little more, both together 1.4 of that.  The workgroups'
// longest, or the work of all, whichever is more; what they begin and end with; for parts the join, 5, and their way to memory and back at 4 TB/s.
//   1 part, 1 group | 1 part, 2 groups | best parts, groups, us: 256 tokens, 32 heads of 128: 12.3, 9.7; 512: 17.9, 13.0; 1024 (8 key heads): 28.3, 25.7; 1536: 41.2, 48.1; 2048: 54.8, 71.6;
//   128 of 2048: 48.5, 29.8, (4, 2) 20.2; 512 of 8192: 175, 107, (4, 1) 82.6; 63 of 32063: (8, 1) 95, (16, 1) 58, (32, 1) 56, (48, 1) 66; 256 of 4096, heads of 64: 59.9, 36.5, (4, 2) 18.1.
// `times`: a tile of the queries' gradient, which has no groups, takes 1.5 times as long.
struct Parts { int splits, groups; };
Parts parts_of(const bw_prompt* p, double times = 1., bool may_group = true) {
    const int share = p->q_heads / p->kv_heads, tile = key_tile(p->dim), cus = bw_device_cus();
    const bool two = p->dim <= 128;                                 // workgroups of one group to a CU
    const int64_t of = p->q_starts ? p->sequences : 1, tiles = (p->q_tokens * share + kRows - 1) / kRows;
    const int64_t row_tiles = p->q_starts ? (tiles > p->sequences ? tiles : p->sequences < p->q_tokens ? p->sequences : p->q_tokens) : p->sequences * tiles_of(p, p->q_tokens, share, kRows);
    const double blocks = (double)p->kv_heads * row_tiles;
    // (of packed sequences, whose lengths are not known here, twice the mean)
    int64_t keys = p->q_starts ? (p->k_tokens * 2 + of - 1) / of : p->k_tokens / p->sequences, rows = p->q_tokens / p->sequences;
    if (keys > p->k_tokens) keys = p->k_tokens;
    auto few = [&](int64_t n) { return n < p->k_tokens ? n : p->k_tokens; };
    const int64_t reach = p->window ? few(p->window) + few(p->sinks) + kRows / share + 2 : keys;
    const bool all = reach >= keys;
    if (!all) keys = reach;
    const double longest = (double)((keys + tile - 1) / tile), mean = all && keys > 0 ? longest * (1. - 0.5 * (rows < keys ? rows : keys) / keys) : longest;
    const double one = times * (p->dim <= 64 ? 0.9 : p->dim <= 96 ? 1.36 : two ? 1.5 : 1.7);
    Parts best = {1, 1};
    double least = 0.;
    for (int groups = 1; groups <= (may_group ? 2 : 1); groups++)
        for (int s = 1; s <= 64 && (s == 1 || s * 2 * groups <= longest); s *= 2) {
            const bool share_cu = groups == 1 && two && blocks * s > cus;
            const double rounds = groups * blocks * s / (cus * (groups == 1 && two ? 2 : 1));
            const double last = longest / (s * groups) * one * (share_cu ? 1.05 : 1.), work = mean * blocks / cus * one * (share_cu ? 0.7 : 1.);
            double time = (last > work ? last : work) + (groups == 1 ? 4. + (rounds > 1. ? rounds : 1.) : 2.5 + 4.5 * (rounds > 1. ? rounds : 1.));
            if (s > 1) time += 5. + (double)p->q_tokens * p->q_heads * p->dim * 8. * s / 4e6;
            const bool plain = s == 1 && groups == 1;
            if (plain || time < least) {
                best = Parts{s, groups};
                least = plain ? 0.95 * time : time;                  // (anything else where it gains something)
            }
        }
    return best;
}

// Pieces of the keys' and values' gradients for each CU, about, over all heads.  All gradients of 8192 tokens, 32 and 8 heads of 128: 1 2182 us, 2 2134, 3 2205, 4 2199; with a window of 1024
// 625, 622, 668, 659.  Of heads up to 64 a CU holds more workgroups at once (8192 tokens, 16 and 4 heads of 64: 1 766 us, 2 701, 3 658, 4 648, 6 640; of 1000 tokens 63, 55, 56, 38, 38).
constexpr int pieces_per_cu(int dim) { return dim <= 64 ? 4 : 2; }

// How the gradients' work is cut, and where their workspace has what (bytes).
struct GradPlan {
    int target;                                  // pieces of a head; 0: every tile of keys is one
    int64_t pieces, parts, joins;                // at most
    int q_splits;                                // parts of a row's keys, for the queries' gradient
    size_t delta, plan, parts_at, q_parts, q_left, all;
};
GradPlan grad_plan(const bw_prompt* p) {
    const int64_t share = p->q_heads / p->kv_heads, seq_q = p->q_tokens / (p->q_starts ? 1 : p->sequences);
    const int tile = key_tile(p->dim);
    const int64_t row_tiles = (seq_q * share + tile - 1) / tile, sequences = p->q_starts ? p->sequences + 2 : p->sequences;
    const int64_t key_tiles = p->q_starts ? p->k_tokens / kGradKeys + sequences : p->sequences * tiles_of(p, p->k_tokens, 1, kGradKeys);
    GradPlan g = {};
    auto room = [&](size_t bytes) {
        const size_t at = g.all;
        g.all += (bytes + 15) / 16 * 16;
        return at;
    };
    g.delta = room((size_t)(p->q_tokens * p->q_heads) * sizeof(float));
    g.q_splits = p->q_tokens > 0 ? parts_of(p, 1.5, false).splits : 1;
    if (g.q_splits > 1) {
        g.q_parts = room((size_t)(p->q_tokens * p->q_heads) * g.q_splits * p->dim * sizeof(float));
        g.q_left = room((size_t)(p->q_tokens * p->q_heads) * g.q_splits * sizeof(float));
    }
    if (row_tiles > 2 * kLeastTiles && p->k_tokens > 0) {
        g.target = (int)(((int64_t)bw_device_cus() * pieces_per_cu(p->dim) + p->kv_heads - 1) / p->kv_heads);
        // (a tile of keys with n of all U tiles of rows is cut into at most n / size, rounded up; size is at least U / target and kLeastTiles.  One that is up to a third longer stays whole)
        g.pieces = key_tiles + g.target;
        const int64_t most = key_tiles * ((row_tiles + kLeastTiles - 1) / kLeastTiles);
        g.parts = 2 * (int64_t)g.target < most ? 2 * g.target : most;
        g.joins = g.parts / 2 < key_tiles ? g.parts / 2 : key_tiles;
        g.plan = room(sizeof(KeyPlan) + 8);
        room((size_t)g.pieces * sizeof(Piece));
        room((size_t)g.joins * sizeof(KeyJoin));
        room((size_t)sequences * sizeof(int));
        g.parts_at = room((size_t)g.parts * p->kv_heads * kGradKeys * 2 * p->dim * sizeof(float));
    }
    return g;
}

}  // namespace

extern "C" size_t bw_prompt_attention_workspace_bytes(const bw_prompt* p) {
    if (prompt_check(p, BW_F16) != BW_OK || p->q_tokens == 0) return 0;
    const int splits = parts_of(p).splits;
    return splits > 1 ? (size_t)(p->q_tokens * p->q_heads) * splits * (p->dim + 2) * sizeof(float) : 0;
}

extern "C" int bw_prompt_attention(const bw_prompt* p, int act_dtype, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                                   const void* v, int64_t v_row, int64_t v_head, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    if (int st = prompt_check(p, act_dtype)) return st;
    if (p->q_tokens == 0) return BW_OK;
    if (!q || !out || (p->k_tokens > 0 && (!k || !v))) return BW_EINVAL;
    if (!bw_aligned(q, 16) || !bw_aligned(k, 16) || !bw_aligned(v, 16) || !bw_aligned(out, 16) || !bw_aligned(lse, 4) || (q_row | q_head | k_row | k_head | v_row | v_head) % 8)
        return BW_EALIGN;
    // (a row's place in its tile of 64 is 32 bits of bytes)
    if (k_row < 0 || v_row < 0 || k_row >= 1 << 24 || v_row >= 1 << 24) return BW_EUNSUPPORTED;
    PromptArgs a = args_of(p);
    a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
    a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head; a.v_row = v_row; a.v_head = v_head;
    a.out = (uint16_t*)out;
    a.lse = lse;
    const Parts parts = parts_of(p);
    a.set_splits(parts.splits);
    const int64_t tiles = tiles_of(p, p->q_tokens, a.share, kRows / parts.groups), grid = tiles * a.combos * a.splits;
    if (grid >= (int64_t)1 << 24) return BW_EUNSUPPORTED;
    a.set_tiles((uint32_t)tiles);
    const size_t bytes = bw_prompt_attention_workspace_bytes(p);
    if (bytes) {
        if (!workspace || workspace_bytes < bytes) return BW_EWORKSPACE;
        if (!bw_aligned(workspace, 16)) return BW_EALIGN;
        a.partial = (float*)workspace;
    }
    const hipStream_t st = (hipStream_t)stream;
    if (int failed = act_dtype == BW_F16 ? bw_launch_prompt_f16(a, (uint32_t)grid, parts.groups, st) : bw_launch_prompt_bf16(a, (uint32_t)grid, parts.groups, st)) return failed;
    if (a.splits > 1) {
        const int threads = p->dim / 4;
        const uint32_t rows = (uint32_t)(p->q_tokens * p->q_heads), per = 256 / threads;
        if (act_dtype == BW_F16) hipLaunchKernelGGL(prompt_join_kernel<BW_F16>, dim3((rows + per - 1) / per), dim3(256), 0, st, a, threads, rows);
        else hipLaunchKernelGGL(prompt_join_kernel<BW_BF16>, dim3((rows + per - 1) / per), dim3(256), 0, st, a, threads, rows);
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    return BW_OK;
}

extern "C" size_t bw_prompt_attention_grad_workspace_bytes(const bw_prompt* p) {
    if (prompt_check(p, BW_F16) != BW_OK) return 0;
    return grad_plan(p).all;
}

extern "C" int bw_prompt_attention_grad(const bw_prompt* p, int act_dtype, const void* grad, int64_t grad_row, int64_t grad_head, const void* q, int64_t q_row,
                                        int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const void* out,
                                        const float* lse, void* q_grad, void* k_grad, void* v_grad, void* workspace, size_t workspace_bytes, void* stream) {
    if (int st = prompt_check(p, act_dtype)) return st;
    if (p->q_tokens > 0 && (!grad || !q || !out || !lse)) return BW_EINVAL;
    if (p->k_tokens > 0 && (!k || !v)) return BW_EINVAL;
    if (!bw_aligned(grad, 16) || !bw_aligned(q, 16) || !bw_aligned(k, 16) || !bw_aligned(v, 16) || !bw_aligned(out, 16) || !bw_aligned(lse, 4) || !bw_aligned(q_grad, 16) ||
        !bw_aligned(k_grad, 16) || !bw_aligned(v_grad, 16) || (grad_row | grad_head | q_row | q_head | k_row | k_head | v_row | v_head) % 8)
        return BW_EALIGN;
    const int64_t share = p->q_heads / p->kv_heads;
    for (int64_t row : {k_row, v_row, q_row, grad_row})
        if (row < 0 || row >= 1 << 24) return BW_EUNSUPPORTED;
    // (a row's place in a tile of rows of a key head's query heads is 32 bits of bytes)
    for (auto [row, head] : {std::pair<int64_t, int64_t>{q_row, q_head}, {grad_row, grad_head}})
        if (head < 0 || head >= (int64_t)1 << 30 || (share - 1) * head + 65 * row >= (int64_t)1 << 31) return BW_EUNSUPPORTED;
    const bool keys = (k_grad || v_grad) && p->k_tokens > 0;
    if (p->q_tokens == 0 && !keys) return BW_OK;
    // (without rows a key's gradients are zeros, whichever sequence it is of: those of one sequence)
    bw_prompt one = *p;
    if (p->q_tokens == 0) {
        one.sequences = 1;
        one.q_starts = one.k_starts = nullptr;
        p = &one;
    }
    const GradPlan plan = grad_plan(p);
    // Workgroups are counted with 31 bits: more than twice as many as any call has that the forward takes, which has fewer than 2^24, a tile of each sequence and key head at least.
    const int64_t combos = p->kv_heads * (int64_t)(p->q_starts ? 1 : p->sequences), key_tiles = tiles_of(p, p->k_tokens, 1, kGradKeys);
    const int64_t row_tiles = p->q_tokens > 0 ? tiles_of(p, p->q_tokens, (int)share, kRows) : 0;
    const int q_splits = q_grad || k_grad ? plan.q_splits : 1;      // (dV alone needs neither dQ nor delta)
    const int64_t row_grid = row_tiles * combos * q_splits, key_grid = !keys ? 0 : plan.target ? plan.pieces * p->kv_heads : key_tiles * combos;
    if (row_grid >= (int64_t)1 << 30 || key_grid >= (int64_t)1 << 30) return BW_EUNSUPPORTED;
    if (plan.all) {
        if (!workspace || workspace_bytes < plan.all) return BW_EWORKSPACE;
        if (!bw_aligned(workspace, 16)) return BW_EALIGN;
    }
    PromptGradArgs g = {};
    g.p = args_of(p);
    PromptArgs& a = g.p;
    a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
    a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head; a.v_row = v_row; a.v_head = v_head;
    a.lse = const_cast<float*>(lse);
    g.grad = (const uint16_t*)grad; g.grad_row = grad_row; g.grad_head = grad_head;
    g.result = (const uint16_t*)out;
    g.q_grad = (uint16_t*)q_grad; g.k_grad = (uint16_t*)k_grad; g.v_grad = (uint16_t*)v_grad;
    g.delta = (float*)workspace;
    a.set_splits(q_splits);
    g.exact = q_grad || k_grad;                                     // (the same for dK, whichever other gradients are wanted)
    g.q_parts = a.splits > 1 ? (float*)((char*)workspace + plan.q_parts) : nullptr;
    g.q_left = a.splits > 1 ? (float*)((char*)workspace + plan.q_left) : nullptr;
    g.plain_scale = p->scale;
    PromptGrids grids = {};
    grids.rows = (uint32_t)row_grid;
    grids.row_tiles = (uint32_t)row_tiles;
    if (keys) {
        grids.keys = (uint32_t)(k_grad && v_grad ? 2 * key_grid : key_grid);
        grids.key_tiles = (uint32_t)key_tiles;
        if (plan.target) {
            grids.joins = (uint32_t)plan.joins;
            char* at = (char*)workspace + plan.plan;
            auto next = [&](size_t bytes) {
                char* here = at;
                at += (bytes + 15) / 16 * 16;
                return here;
            };
            g.target = plan.target;
            g.room = (int)plan.pieces; g.parts_room = (int)plan.parts; g.joins_room = (int)plan.joins;
            g.plan = (KeyPlan*)next(sizeof(KeyPlan) + 8);
            g.pieces = (Piece*)next((size_t)plan.pieces * sizeof(Piece));
            g.joins = (KeyJoin*)next((size_t)plan.joins * sizeof(KeyJoin));
            g.tiles_before = (int*)at;
            g.parts = (float*)((char*)workspace + plan.parts_at);
        }
    }
    const hipStream_t st = (hipStream_t)stream;
    return act_dtype == BW_F16 ? bw_launch_prompt_grad_f16(g, grids, st) : bw_launch_prompt_grad_bf16(g, grids, st);
}
