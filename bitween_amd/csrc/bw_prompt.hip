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
    // (scale 0: all scores that are numbers weigh the same, and hidden ones, minus infinity, stay hidden)
    const float scale = __builtin_fabsf(p->scale) * 1.44269504088896340736f;
    a.scale = scale < 1e-38f ? 1e-38f : scale;
    return a;
}

int key_tile(int dim) { return dim > 128 ? 32 : 64; }

// Parts that the keys of a tile of rows are cut into: the number for which the longest workgroup (or, in several rounds, the mean of all), the second launch and the parts' way
// through memory take the least together.  In microseconds, as measured: a tile of keys takes a workgroup 0.9 (heads of 64), 1.5 (128) and 2 (256, of half the keys), 1.4 times that
// where two share a CU; the join 5, and its parts, written and read, go at 4 TB/s.  512 tokens of 8192, 32 and 8 heads of 128: 1 part 193 us, 2 110, 3 100, 4 88; 63 of 32063: 8 parts 106 us,
// 16 63, 32 59, 48 70; 1024 tokens alone: 1 part 31 us, 2 41; 256 of 4096, heads of 64: 1 part 62 us, 4 25, 8 20, 16 26.  `times`: a tile of the queries' gradient takes 1.25 times as long.
int splits_of(const bw_prompt* p, double times = 1.) {
    const int share = p->q_heads / p->kv_heads, tile = key_tile(p->dim), cus = bw_device_cus(), resident = cus * (p->dim > 128 ? 1 : 2);
    const int64_t of = p->q_starts ? p->sequences : 1, tiles = (p->q_tokens * share + kRows - 1) / kRows;
    const int64_t row_tiles = p->q_starts ? (tiles > p->sequences ? tiles : p->sequences < p->q_tokens ? p->sequences : p->q_tokens) : p->sequences * tiles_of(p, p->q_tokens, share, kRows);
    const double blocks = (double)p->kv_heads * row_tiles;
    // (of packed sequences, whose lengths are not known here, twice the mean)
    int64_t keys = p->q_starts ? (p->k_tokens * 2 + of - 1) / of : p->k_tokens / p->sequences, rows = p->q_tokens / p->sequences;
    if (keys > p->k_tokens) keys = p->k_tokens;
    const int64_t reach = p->window ? p->window + p->sinks + kRows / share + 2 : keys;
    const bool all = reach >= keys;
    if (!all) keys = reach;
    const double longest = (double)((keys + tile - 1) / tile), mean = all && keys > 0 ? longest * (1. - 0.5 * (rows < keys ? rows : keys) / keys) : longest;
    const double one = times * (p->dim > 128 ? 2.0 : 0.3 + p->dim * 0.0094);
    int best = 1;
    double least = 0.;
    for (int s = 1; s <= 64 && (s == 1 || s * 2 <= longest); s++) {
        const double rounds = blocks * s / resident, tiles_each = rounds > 1. && mean * rounds > longest ? mean * rounds : longest;
        const double time = tiles_each / s * one * (blocks * s > cus && resident > cus ? 1.4 : 1.) + (s > 1 ? 5. + (double)p->q_tokens * p->q_heads * p->dim * 8. * s / 4e6 : 0.);
        if (s == 1 || time < least) {
            best = s;
            least = s == 1 ? 0.9 * time : time;                      // (parts where they gain a tenth at least)
        }
    }
    return best;
}

// How the gradients' work is cut, and where their workspace has what (bytes).
// About, over all heads (8192 tokens, 32 and 8 heads of 128, gradients of keys and values: 1 1549 us, 2 1479, 3 1495, 4 1513; with a window of 1024 451, 444, 512, 483; 2048 tokens 149, 153,
// 162, 160).  Of heads up to 64 a CU holds more workgroups at once (16 and 4 heads of 64: 2 480 us, 4 438).
constexpr int pieces_per_cu(int dim) { return dim <= 64 ? 4 : 2; }
struct GradPlan {
    int target;                                  // pieces of a head; 0: every tile of keys is one
    int64_t pieces, parts, joins;                // at most
    int q_splits;                                // parts of a row's keys, for the queries' gradient
    size_t delta, plan, parts_at, q_parts, all;
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
    g.q_splits = p->q_tokens > 0 ? splits_of(p, 1.25) : 1;
    if (g.q_splits > 1) g.q_parts = room((size_t)(p->q_tokens * p->q_heads) * g.q_splits * p->dim * sizeof(float));
    if (row_tiles > 2 * kLeastTiles && p->k_tokens > 0) {
        g.target = (int)(((int64_t)bw_device_cus() * pieces_per_cu(p->dim) + p->kv_heads - 1) / p->kv_heads);
        // (a tile of n among U tiles of rows is cut into n / size rounded up, size at least U / target and kLeastTiles)
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
    const int splits = splits_of(p);
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
    a.set_splits(splits_of(p));
    const int64_t tiles = tiles_of(p, p->q_tokens, a.share, kRows), grid = tiles * a.combos * a.splits;
    if (grid >= (int64_t)1 << 24) return BW_EUNSUPPORTED;
    a.set_tiles((uint32_t)tiles);
    const size_t bytes = bw_prompt_attention_workspace_bytes(p);
    if (bytes) {
        if (!workspace || workspace_bytes < bytes) return BW_EWORKSPACE;
        if (!bw_aligned(workspace, 16)) return BW_EALIGN;
        a.partial = (float*)workspace;
    }
    const hipStream_t st = (hipStream_t)stream;
    if (int failed = act_dtype == BW_F16 ? bw_launch_prompt_f16(a, (uint32_t)grid, st) : bw_launch_prompt_bf16(a, (uint32_t)grid, st)) return failed;
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
    const GradPlan plan = grad_plan(p);
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
    a.set_splits(q_grad ? plan.q_splits : 1);
    g.q_parts = a.splits > 1 ? (float*)((char*)workspace + plan.q_parts) : nullptr;
    g.plain_scale = p->scale;
    PromptGrids grids = {};
    if (p->q_tokens > 0) {
        const int64_t tiles = tiles_of(p, p->q_tokens, a.share, kRows), grid = tiles * a.combos * a.splits;
        if (grid >= (int64_t)1 << 24) return BW_EUNSUPPORTED;
        grids.rows = (uint32_t)grid;
        grids.row_tiles = (uint32_t)tiles;
    }
    if (keys) {
        const int64_t tiles = tiles_of(p, p->k_tokens, 1, kGradKeys), grid = plan.target ? plan.pieces * p->kv_heads : tiles * a.combos;
        if (grid >= (int64_t)1 << 23 || plan.joins * p->kv_heads >= (int64_t)1 << 22) return BW_EUNSUPPORTED;
        grids.keys = (uint32_t)(k_grad && v_grad ? 2 * grid : grid);
        grids.key_tiles = (uint32_t)tiles;
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
