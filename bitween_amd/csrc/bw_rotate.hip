// Rotation of queries and keys by the angle of their token's position, with the norm of each head in the same pass, and its gradients.
//
// Which values a thread has, and its angles, are in bw_rotate.h.
//
// Gradients, with n = x r, r = rsqrt(mean(x^2) + eps) and g' the incoming gradient turned back:
//   dx = r (g' w - n mean(g' w n)),  dw = sum over tokens and heads of g' n
// The sum of dw is taken by every thread over the heads it meets, by its workgroup through LDS and by a second kernel over the workgroups,
// each in a fixed order.
//
// One pass over memory, a dozen float32 operations a value: launch-bound up to a few hundred tokens (one token 2.3 us as a graph), HBM and, as every head
// loads its token's cosines and sines, the L2 beyond: 2048 tokens of 32 and 8 heads of 128 in bfloat16 with both norms take 11 us (42 MB, 3.8 TB/s),
// their gradients 17 (63 MB) and 4 for the sum; torch copies 21 MB in 7 us.  By three axes: 1024 tokens without norms 8 us, 4095 with norms 19 (84 MB, 4.4 TB/s), their gradients 37 (126 MB, 3.4 TB/s:
// the forward asks for the next head's values while it has one, they ask for a head's when they need them)
// and 4, 16384 without 73 (335 MB, 4.6 TB/s).
#include "bw_rotate.h"

namespace {

// One head of a thread: loaded, normed, turned, stored.
template <int DT, int CH> BW_DEV void rotate_head(const RotateArgs& a, const Raw<CH>& raw1, const Raw<CH>& raw2, const Angle<CH>& angle, int token, int head, bool live, bool kept, bool turns,
                                                  int first, int second) {
    const bool is_k = head >= a.q_heads;
    if (is_k) head -= a.q_heads;
    float x[CH], y[CH];
    widen_raw<DT, CH>(raw1, x);
    widen_raw<DT, CH>(raw2, y);
    if (a.q_weight || a.k_weight) {
        const void* weight = is_k ? a.k_weight : a.q_weight;
        float ss = 0.f;
        if (live) {
#pragma unroll
            for (int j = 0; j < CH; j++) ss += x[j] * x[j] + y[j] * y[j];
        }
        ss = head_sum(ss, a.lane_shift);
        if (weight) {
            const float r = rsqrtf(ss / (float)a.dim + a.eps);
            float w[CH];
            load_weight<DT, CH>(weight, a.weight_f32, first, w);
#pragma unroll
            for (int j = 0; j < CH; j++) x[j] = x[j] * r * w[j];
            load_weight<DT, CH>(weight, a.weight_f32, second, w);
#pragma unroll
            for (int j = 0; j < CH; j++) y[j] = y[j] * r * w[j];
        }
    }
    if (!kept) {
#pragma unroll
        for (int j = 0; j < CH; j++) x[j] = y[j] = 0.f;
    } else if (turns) {
        angle.template turn<1>(x, y);
    }
    if (!live) return;
    uint16_t* dst = is_k ? a.k_out + ((int64_t)token * a.k_heads + head) * a.dim : a.q_out + ((int64_t)token * a.q_heads + head) * a.dim;
    store_chunk<DT, CH>(dst + first, x);
    store_chunk<DT, CH>(dst + second, y);
}

template <int DT, int CH>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a) {
    const uint32_t heads = (uint32_t)(a.q_heads + a.k_heads), item = (blockIdx.x * 256 + threadIdx.x) >> a.lane_shift;
    const int lane = (int)threadIdx.x & ((1 << a.lane_shift) - 1);
    const bool live = item < (uint32_t)a.T * heads && lane < a.lanes;
    const uint32_t it = live ? item : 0;
    const int token = (int)(it / heads), head = (int)(it - (uint32_t)token * heads);
    int first, second;
    bool turns;
    chunks_of<CH>(a, live ? lane : 0, first, second, turns);
    const uint16_t* src = head >= a.q_heads ? a.k + token * a.k_row + (head - a.q_heads) * a.k_head : a.q + token * a.q_row + head * a.q_head;
    const Position<false> pos(a, token);
    const Raw<CH> raw1 = load_raw<CH>(src + first), raw2 = load_raw<CH>(src + second);
    Angle<CH> angle;
    if (pos.kept && turns) angle.load(a, pos, first);
    rotate_head<DT, CH>(a, raw1, raw2, angle, token, head, live, pos.kept, turns, first, second);
}

// Positions of several axes: the angles come from as many rows of the tables as there are axes, so that a thread keeps them for several heads of its token, a.slices apart
// (4095 tokens of 32 and 8 heads of 128 with norms, three interleaved axes: 26.6 us with one head).
template <int DT, int CH>
__global__ __launch_bounds__(256) void rotate_axes_kernel(RotateArgs a) {
    const uint32_t heads = (uint32_t)(a.q_heads + a.k_heads), item = (blockIdx.x * 256 + threadIdx.x) >> a.lane_shift;
    const int lane = (int)threadIdx.x & ((1 << a.lane_shift) - 1);
    const bool live = item < (uint32_t)a.T * a.slices && lane < a.lanes;
    const uint32_t it = live ? item : 0;
    const int token = (int)(it / a.slices);
    int first, second;
    bool turns;
    chunks_of<CH>(a, live ? lane : 0, first, second, turns);
    const Position<true> pos(a, token);
    auto source = [&](uint32_t head) { return (int)head >= a.q_heads ? a.k + token * a.k_row + ((int)head - a.q_heads) * a.k_head : a.q + token * a.q_row + (int)head * a.q_head; };
    uint32_t head = it - (uint32_t)token * a.slices;
    const uint16_t* src = source(head);
    Raw<CH> raw1 = load_raw<CH>(src + first), raw2 = load_raw<CH>(src + second);
    Angle<CH> angle;
    if (pos.kept && turns) angle.load(a, pos, first);
    for (;;) {
        const uint32_t next = head + a.slices;
        const bool more = next < heads;
        src = source(more ? next : head);
        const Raw<CH> next1 = load_raw<CH>(src + first), next2 = load_raw<CH>(src + second);
        rotate_head<DT, CH>(a, raw1, raw2, angle, token, (int)head, live, pos.kept, turns, first, second);
        if (!more) return;
        head = next;
        raw1 = next1;
        raw2 = next2;
    }
}

// One block serves the queries' heads or the keys', 256 >> lane_shift at a time.
template <int DT, int CH, bool AXES>
__global__ __launch_bounds__(256) void rotate_grad_kernel(RotateArgs a) {
    __shared__ float sums[256 * 2 * CH];
    const bool is_k = (int)blockIdx.x >= a.q_blocks;
    const uint32_t heads = (uint32_t)(is_k ? a.k_heads : a.q_heads), per_block = 256u >> a.lane_shift, items = (uint32_t)a.T * (AXES ? (is_k ? a.k_slices : a.slices) : heads);
    const uint32_t block = is_k ? blockIdx.x - a.q_blocks : blockIdx.x, blocks = is_k ? gridDim.x - a.q_blocks : a.q_blocks;
    const int lane = (int)threadIdx.x & ((1 << a.lane_shift) - 1);
    int first, second;
    bool turns;
    chunks_of<CH>(a, lane < a.lanes ? lane : 0, first, second, turns);
    const void* weight = is_k ? a.k_weight : a.q_weight;
    const uint16_t* xs = is_k ? a.k : a.q;
    const uint16_t* gs = is_k ? a.gk : a.gq;
    const int64_t x_row = is_k ? a.k_row : a.q_row, x_head = is_k ? a.k_head : a.q_head;
    const int64_t g_row = is_k ? a.gk_row : a.gq_row, g_head = is_k ? a.gk_head : a.gq_head;
    uint16_t* out = is_k ? a.k_out : a.q_out;
    float w1[CH] = {}, w2[CH] = {}, d1[CH] = {}, d2[CH] = {};
    if (weight) {
        load_weight<DT, CH>(weight, a.weight_f32, first, w1);
        load_weight<DT, CH>(weight, a.weight_f32, second, w2);
    }
    Angle<CH> angle;
    bool kept = false;
    // (the same number of rounds for every thread of the block: all of them take part in the sums; positions of several axes: heads of a token, a.slices or a.k_slices apart, one after the
    // other, which share their angles)
    for (uint32_t base = block * per_block, turn = 0; base < items;) {
        const uint32_t item = base + (threadIdx.x >> a.lane_shift);
        const uint32_t per_token = AXES ? (is_k ? a.k_slices : a.slices) : heads, it0 = item < items && lane < a.lanes ? item : 0;
        const int token = (int)(it0 / per_token), head0 = (int)(it0 - (uint32_t)token * per_token + turn * per_token);
        const bool live = item < items && lane < a.lanes && (!AXES || head0 < (int)heads);
        const int head = live ? head0 : 0;
        if (!AXES || turn == 0) {
            const Position<AXES> pos(a, token);
            kept = pos.kept;
            if (kept && turns) angle.load(a, pos, first);
        }
        if (AXES && (turn + 1) * per_token < heads) turn++;
        else {
            turn = 0;
            base += blocks * per_block;
        }
        const uint16_t* g = gs + token * g_row + head * g_head;
        const uint16_t* in = xs + token * x_row + head * x_head;
        const Raw<CH> g1 = load_raw<CH>(g + first), g2 = load_raw<CH>(g + second);
        Raw<CH> x1 = {}, x2 = {};
        if (weight) {
            x1 = load_raw<CH>(in + first);
            x2 = load_raw<CH>(in + second);
        }
        float x[CH], y[CH];
        widen_raw<DT, CH>(g1, x);
        widen_raw<DT, CH>(g2, y);
        if (!kept) {
#pragma unroll
            for (int j = 0; j < CH; j++) x[j] = y[j] = 0.f;
        } else if (turns) {
            angle.template turn<-1>(x, y);
        }
        if (weight) {
            float n1[CH], n2[CH], ss = 0.f, dot = 0.f;
            widen_raw<DT, CH>(x1, n1);
            widen_raw<DT, CH>(x2, n2);
            if (live) {
#pragma unroll
                for (int j = 0; j < CH; j++) ss += n1[j] * n1[j] + n2[j] * n2[j];
            }
            ss = head_sum(ss, a.lane_shift);
            const float r = rsqrtf(ss / (float)a.dim + a.eps);
#pragma unroll
            for (int j = 0; j < CH; j++) {
                n1[j] *= r;
                n2[j] *= r;
                if (live && kept) {
                    d1[j] += x[j] * n1[j];
                    d2[j] += y[j] * n2[j];
                    dot += x[j] * w1[j] * n1[j] + y[j] * w2[j] * n2[j];
                }
            }
            dot = head_sum(dot, a.lane_shift) / (float)a.dim;
#pragma unroll
            for (int j = 0; j < CH; j++) {
                x[j] = kept ? r * (x[j] * w1[j] - n1[j] * dot) : 0.f;
                y[j] = kept ? r * (y[j] * w2[j] - n2[j] * dot) : 0.f;
            }
        }
        if (live) {
            uint16_t* dst = out + ((int64_t)token * heads + head) * a.dim;
            store_chunk<DT, CH>(dst + first, x);
            store_chunk<DT, CH>(dst + second, y);
        }
    }
    if (!weight || !a.partial) return;                        // uniform over the block
#pragma unroll
    for (int j = 0; j < CH; j++) {
        sums[threadIdx.x * 2 * CH + j] = d1[j];
        sums[threadIdx.x * 2 * CH + CH + j] = d2[j];
    }
    __syncthreads();
    for (int at = (int)threadIdx.x; at < a.lanes * 2 * CH; at += 256) {
        const int l = at / (2 * CH), j = at - l * 2 * CH;
        float s = 0.f;
        for (uint32_t i = 0; i < per_block; i++) s += sums[((i << a.lane_shift) + l) * 2 * CH + j];
        int f, g;
        bool t;
        chunks_of<CH>(a, l, f, g, t);
        a.partial[(int64_t)blockIdx.x * a.dim + (j < CH ? f + j : g + j - CH)] = s;
    }
}

// dw = the sum of its blocks' rows: one workgroup for 32 columns of a weight, 128 rows at a time, four of a thread under way (32 rows at a time: 4.9 us
// for 819 and 205 rows).
template <int DT>
__global__ __launch_bounds__(1024) void weight_grad_kernel(const float* partial, int dim, int q_blocks, int blocks, void* q_grad, void* k_grad, int f32) {
    __shared__ f4 sums[128][8];
    const bool is_k = blockIdx.y == 1;
    void* out = is_k ? k_grad : q_grad;
    if (!out) return;
    const int to = is_k ? blocks : q_blocks, x = (int)threadIdx.x & 7, y = (int)threadIdx.x >> 3, d = (int)blockIdx.x * 32 + 4 * x;
    f4 s = {0.f, 0.f, 0.f, 0.f};
    if (d < dim)
        for (int b = (is_k ? q_blocks : 0) + y; b < to; b += 512) {
            f4 v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = b + 128 * i < to ? *reinterpret_cast<const f4*>(partial + (int64_t)(b + 128 * i) * dim + d) : f4{0.f, 0.f, 0.f, 0.f};
            s += (v[0] + v[1]) + (v[2] + v[3]);
        }
    sums[y][x] = s;
    __syncthreads();
    if (y < 8) {
#pragma unroll
        for (int i = 1; i < 16; i++) s += sums[y + 8 * i][x];
    }
    __syncthreads();
    if (y < 8) sums[y][x] = s;
    __syncthreads();
    if (y || d >= dim) return;
#pragma unroll
    for (int i = 1; i < 8; i++) s += sums[i][x];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (f32) ((float*)out)[d + j] = s[j];
        else ((uint16_t*)out)[d + j] = narrow16<DT>(s[j]);
    }
}

// Blocks of the gradient kernel for the queries or the keys: enough to fill the chip together, 1024 in proportion to their heads, so that the
// sums over them stay short (2048 tokens of 32 and 8 heads of 128, forward and backward: 30.2 us; with 768 30.5, 1536 31.9, 2048 33.1).
int grad_blocks(const bw_heads* h, int heads) {
    const int per_block = 256 >> bw_log2(h->dim / (2 * chunk_of(h))), all = h->q_heads + h->k_heads;
    const int64_t want = (h->tokens * heads + per_block - 1) / per_block, most = ((int64_t)1024 * heads + all - 1) / all;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

int rotate(const bw_heads* h, const bw_axes* x, int act_dtype, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, void* q_out,
           void* k_out, void* stream) {
    if (int st = heads_check(h, act_dtype)) return st;
    if (h->tokens == 0) return BW_OK;
    if (!q || !k || !q_out || !k_out) return BW_EINVAL;
    if (!bw_aligned(q, 16) || !bw_aligned(k, 16) || !bw_aligned(q_out, 16) || !bw_aligned(k_out, 16) || (q_row | q_head | k_row | k_head) % 8) return BW_EALIGN;
    RotateArgs a = rotate_args(h, x);
    a.q = (const uint16_t*)q; a.k = (const uint16_t*)k;
    a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head;
    a.q_out = (uint16_t*)q_out; a.k_out = (uint16_t*)k_out;
    // In several launches where a head's lanes, filled up to a power of two, would pass the 2^32 threads of one.
    const int64_t heads = h->q_heads + h->k_heads, per_block = 256 >> a.lane_shift, most = (((int64_t)1 << 32) - 256) / (heads << a.lane_shift);
    for (int64_t at = 0; at < h->tokens; at += most) {
        a.T = (int)(h->tokens - at < most ? h->tokens - at : most);
        a.slices = x ? (uint32_t)slices_of(a, (int)heads) : (uint32_t)heads;
        const dim3 grid((unsigned)(((int64_t)a.T * a.slices + per_block - 1) / per_block)), block(256);
#define BW_ROTATE(DT, CH) \
    if (act_dtype == DT && chunk_of(h) == CH && x) hipLaunchKernelGGL((rotate_axes_kernel<DT, CH>), grid, block, 0, (hipStream_t)stream, a); \
    else if (act_dtype == DT && chunk_of(h) == CH) hipLaunchKernelGGL((rotate_kernel<DT, CH>), grid, block, 0, (hipStream_t)stream, a);
        BW_ROTATE(BW_F16, 8) BW_ROTATE(BW_F16, 4) BW_ROTATE(BW_BF16, 8) BW_ROTATE(BW_BF16, 4)
#undef BW_ROTATE
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
        a.positions += a.T;
        a.q += a.T * q_row; a.k += a.T * k_row;
        a.q_out += (int64_t)a.T * h->q_heads * h->dim; a.k_out += (int64_t)a.T * h->k_heads * h->dim;
    }
    return BW_OK;
}

size_t grad_workspace(const bw_heads* h) {
    if (heads_check(h, h && h->weight_dtype == BW_BF16 ? BW_BF16 : BW_F16) != BW_OK || (!h->q_weight && !h->k_weight)) return 0;
    return (size_t)(grad_blocks(h, h->q_heads) + grad_blocks(h, h->k_heads)) * h->dim * sizeof(float);
}

int rotate_grad(const bw_heads* h, const bw_axes* x, int act_dtype, const void* gq, int64_t gq_row, int64_t gq_head, const void* gk, int64_t gk_row, int64_t gk_head,
                const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, void* q_grad, void* k_grad, void* q_weight_grad,
                void* k_weight_grad, void* workspace, size_t workspace_bytes, void* stream) {
    if (int st = heads_check(h, act_dtype)) return st;
    if ((q_weight_grad && !h->q_weight) || (k_weight_grad && !h->k_weight)) return BW_EINVAL;
    if (h->tokens > 0) {
        if (!gq || !gk || !q_grad || !k_grad || (h->q_weight && !q) || (h->k_weight && !k)) return BW_EINVAL;
        if (!bw_aligned(gq, 16) || !bw_aligned(gk, 16) || !bw_aligned(q, 16) || !bw_aligned(k, 16) || !bw_aligned(q_grad, 16) || !bw_aligned(k_grad, 16) ||
            (gq_row | gq_head | gk_row | gk_head) % 8)
            return BW_EALIGN;
        if ((h->q_weight && (q_row | q_head) % 8) || (h->k_weight && (k_row | k_head) % 8)) return BW_EALIGN;
    }
    RotateArgs a = rotate_args(h, x);
    a.gq = (const uint16_t*)gq; a.gk = (const uint16_t*)gk;
    a.gq_row = gq_row; a.gq_head = gq_head; a.gk_row = gk_row; a.gk_head = gk_head;
    a.q = (const uint16_t*)q; a.k = (const uint16_t*)k;
    a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head;
    a.q_out = (uint16_t*)q_grad; a.k_out = (uint16_t*)k_grad;
    a.q_blocks = h->tokens ? grad_blocks(h, h->q_heads) : 0;
    const int blocks = h->tokens ? a.q_blocks + grad_blocks(h, h->k_heads) : 0;
    if (x) {
        // (as many heads to a thread as there would be rounds: each block has about one)
        auto slices = [&](int heads, int of) {
            const int64_t rounds = h->tokens ? ((h->tokens * heads << a.lane_shift) + 256 * (int64_t)of - 1) / (256 * (int64_t)of) : 1;
            const int each = (int)(rounds < 8 ? rounds : 8);
            return (uint32_t)((heads + each - 1) / each);
        };
        a.slices = slices(h->q_heads, a.q_blocks);
        a.k_slices = slices(h->k_heads, blocks - a.q_blocks);
    }
    const bool sums = q_weight_grad || k_weight_grad;
    if (sums && blocks) {
        if (!workspace || workspace_bytes < grad_workspace(h)) return BW_EWORKSPACE;
        if (!bw_aligned(workspace, 16)) return BW_EALIGN;
        a.partial = (float*)workspace;
    }
    if (blocks) {
#define BW_ROTATE(DT, CH) \
    if (act_dtype == DT && chunk_of(h) == CH && x) hipLaunchKernelGGL((rotate_grad_kernel<DT, CH, true>), dim3(blocks), dim3(256), 0, (hipStream_t)stream, a); \
    else if (act_dtype == DT && chunk_of(h) == CH) hipLaunchKernelGGL((rotate_grad_kernel<DT, CH, false>), dim3(blocks), dim3(256), 0, (hipStream_t)stream, a);
        BW_ROTATE(BW_F16, 8) BW_ROTATE(BW_F16, 4) BW_ROTATE(BW_BF16, 8) BW_ROTATE(BW_BF16, 4)
#undef BW_ROTATE
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    if (sums) {                                               // (without tokens: zeros)
        if (act_dtype == BW_F16)
            hipLaunchKernelGGL(weight_grad_kernel<BW_F16>, dim3((h->dim + 31) / 32, 2), dim3(1024), 0, (hipStream_t)stream, a.partial, h->dim, a.q_blocks, blocks, q_weight_grad, k_weight_grad, a.weight_f32);
        else
            hipLaunchKernelGGL(weight_grad_kernel<BW_BF16>, dim3((h->dim + 31) / 32, 2), dim3(1024), 0, (hipStream_t)stream, a.partial, h->dim, a.q_blocks, blocks, q_weight_grad, k_weight_grad, a.weight_f32);
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    return BW_OK;
}

}  // namespace

extern "C" int bw_rotate_heads(const bw_heads* h, int act_dtype, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                               int64_t k_head, void* q_out, void* k_out, void* stream) {
    return rotate(h, nullptr, act_dtype, q, q_row, q_head, k, k_row, k_head, q_out, k_out, stream);
}

extern "C" int bw_rotate_axes(const bw_heads* h, const bw_axes* axes, int act_dtype, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                              int64_t k_head, void* q_out, void* k_out, void* stream) {
    if (int st = axes_check(axes, h ? h->rotary : 0)) return st;
    return rotate(h, axes, act_dtype, q, q_row, q_head, k, k_row, k_head, q_out, k_out, stream);
}

extern "C" size_t bw_rotate_heads_grad_workspace_bytes(const bw_heads* h) { return grad_workspace(h); }

extern "C" int bw_rotate_heads_grad(const bw_heads* h, int act_dtype, const void* gq, int64_t gq_row, int64_t gq_head, const void* gk, int64_t gk_row,
                                    int64_t gk_head, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                                    void* q_grad, void* k_grad, void* q_weight_grad, void* k_weight_grad, void* workspace, size_t workspace_bytes,
                                    void* stream) {
    return rotate_grad(h, nullptr, act_dtype, gq, gq_row, gq_head, gk, gk_row, gk_head, q, q_row, q_head, k, k_row, k_head, q_grad, k_grad, q_weight_grad, k_weight_grad,
                       workspace, workspace_bytes, stream);
}

extern "C" int bw_rotate_axes_grad(const bw_heads* h, const bw_axes* axes, int act_dtype, const void* gq, int64_t gq_row, int64_t gq_head, const void* gk, int64_t gk_row,
                                   int64_t gk_head, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, void* q_grad, void* k_grad,
                                   void* q_weight_grad, void* k_weight_grad, void* workspace, size_t workspace_bytes, void* stream) {
    if (int st = axes_check(axes, h ? h->rotary : 0)) return st;
    return rotate_grad(h, axes, act_dtype, gq, gq_row, gq_head, gk, gk_row, gk_head, q, q_row, q_head, k, k_row, k_head, q_grad, k_grad, q_weight_grad, k_weight_grad,
                       workspace, workspace_bytes, stream);
}
