// Rotation of queries and keys by the angle of their token's position, with the norm of each head in the same pass, and its gradients.
//
// A thread owns CH values of a head and the CH values half a rotation further on, the pairs that turn together (behind the rotated part:
// twice CH neighbours), so that a pair never leaves its thread.  2^lane_shift neighbouring threads hold a head (as many as it needs, filled up
// to a power of two), and the sums that the norm needs go over them with cross-lane shuffles.
//
// Gradients, with n = x r, r = rsqrt(mean(x^2) + eps) and g' the incoming gradient turned back:
//   dx = r (g' w - n mean(g' w n)),  dw = sum over tokens and heads of g' n
// The sum of dw is taken by every thread over the heads it meets, by its workgroup through LDS and by a second kernel over the workgroups,
// each in a fixed order.
//
// One pass over memory, a dozen float32 operations a value: launch-bound up to a few hundred tokens (one token 2.3 us as a graph), HBM and, as every head
// loads its token's cosines and sines, the L2 beyond: 2048 tokens of 32 and 8 heads of 128 in bfloat16 with both norms take 11 us (42 MB, 3.8 TB/s),
// their gradients 17 (63 MB) and 4 for the sum; torch copies 21 MB in 7 us.
#include "bw_cache.h"

namespace {

constexpr int kMaxDim = 256;

struct RotateArgs {
    const uint16_t *q, *k, *gq, *gk;
    int64_t q_row, q_head, k_row, k_head, gq_row, gq_head, gk_row, gk_head;
    uint16_t *q_out, *k_out;                     // rotated heads, or the gradients of the inputs
    const float *cos, *sin;
    const int64_t* positions;
    const void *q_weight, *k_weight;
    float* partial;                              // [blocks][dim]: sums of dw, the queries' blocks first
    int64_t table_rows;
    int T, q_heads, k_heads, dim, half, lanes, lane_shift, weight_f32;
    int q_blocks;                                // gradient: blocks that serve the queries
    float eps;
};

// CH 16-bit values as they come from memory, and as float32.
template <int CH> using Raw = std::conditional_t<CH == 8, u4, u2>;
template <int CH> BW_DEV Raw<CH> load_raw(const uint16_t* p) { return *reinterpret_cast<const Raw<CH>*>(p); }
template <int DT, int CH> BW_DEV void widen_raw(const Raw<CH>& w, float* x) {
#pragma unroll
    for (int j = 0; j < CH; j++) x[j] = widen16<DT>((uint16_t)(w[j / 2] >> (16 * (j & 1))));
}

template <int DT, int CH>
BW_DEV void store_chunk(uint16_t* p, const float* x) {
    uint32_t w[CH / 2];
#pragma unroll
    for (int j = 0; j < CH / 2; j++) w[j] = narrow_pair<DT>(x[2 * j], x[2 * j + 1]);
    if constexpr (CH == 8) *reinterpret_cast<u4*>(p) = u4{w[0], w[1], w[2], w[3]};
    else *reinterpret_cast<u2*>(p) = u2{w[0], w[1]};
}

template <int DT, int CH>
BW_DEV void load_weight(const void* w, int f32, int at, float* x) {
    if (f32) {
#pragma unroll
        for (int j = 0; j < CH; j++) x[j] = ((const float*)w)[at + j];
    } else {
        widen_raw<DT, CH>(load_raw<CH>((const uint16_t*)w + at), x);
    }
}

template <int CH>
BW_DEV void load_floats(const float* p, float* x) {
#pragma unroll
    for (int j = 0; j < CH / 4; j++) {
        const f4 v = *reinterpret_cast<const f4*>(p + 4 * j);
        x[4 * j] = v[0]; x[4 * j + 1] = v[1]; x[4 * j + 2] = v[2]; x[4 * j + 3] = v[3];
    }
}

// The two chunks of lane c of a head, and whether they turn.
template <int CH>
BW_DEV void chunks_of(const RotateArgs& a, int c, int& first, int& second, bool& turns) {
    const int pairs = a.half / CH;
    turns = c < pairs;
    first = turns ? c * CH : 2 * a.half + 2 * (c - pairs) * CH;
    second = turns ? first + a.half : first + CH;
}

// Over the 2^shift lanes of a head, each with the sum: neighbours, pairs, then mirrored halves of 8 and of 16, whose lanes hold the same by then.
template <int CTRL> BW_DEV float from_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
BW_DEV float head_sum(float v, int shift) {
    if (shift > 0) v += from_lane<0xB1>(v);
    if (shift > 1) v += from_lane<0x4E>(v);
    if (shift > 2) v += from_lane<0x141>(v);
    if (shift > 3) v += from_lane<0x140>(v);
    if (shift > 4) v += __shfl_xor(v, 16, 64);
    return v;
}

// cos and sin of a thread's pairs.
template <int CH> struct Angle {
    float c[CH], s[CH];
    BW_DEV void load(const RotateArgs& a, int64_t pos, int first) {
        load_floats<CH>(a.cos + pos * a.half + first, c);
        load_floats<CH>(a.sin + pos * a.half + first, s);
    }
    // SIGN 1: turned by the angle, -1: turned back
    template <int SIGN> BW_DEV void turn(float* x, float* y) const {
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const float u = x[j], v = y[j];
            x[j] = u * c[j] - SIGN * v * s[j];
            y[j] = v * c[j] + SIGN * u * s[j];
        }
    }
};

template <int DT, int CH>
__global__ __launch_bounds__(256) void rotate_kernel(RotateArgs a) {
    const uint32_t heads = (uint32_t)(a.q_heads + a.k_heads), item = (blockIdx.x * 256 + threadIdx.x) >> a.lane_shift;
    const int lane = (int)threadIdx.x & ((1 << a.lane_shift) - 1);
    const bool live = item < (uint32_t)a.T * heads && lane < a.lanes;
    const uint32_t it = live ? item : 0;
    const int token = (int)(it / heads);
    int head = (int)(it - (uint32_t)token * heads);
    const bool is_k = head >= a.q_heads;
    if (is_k) head -= a.q_heads;
    int first, second;
    bool turns;
    chunks_of<CH>(a, live ? lane : 0, first, second, turns);
    const uint16_t* src = is_k ? a.k + token * a.k_row + head * a.k_head : a.q + token * a.q_row + head * a.q_head;
    const int64_t pos = a.positions[token];
    float x[CH], y[CH];
    widen_raw<DT, CH>(load_raw<CH>(src + first), x);
    widen_raw<DT, CH>(load_raw<CH>(src + second), y);
    const bool kept = pos >= 0 && pos < a.table_rows;
    Angle<CH> angle;
    if (kept && turns) angle.load(a, pos, first);
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

// One block serves the queries' heads or the keys', 256 >> lane_shift at a time.
template <int DT, int CH>
__global__ __launch_bounds__(256) void rotate_grad_kernel(RotateArgs a) {
    __shared__ float sums[256 * 2 * CH];
    const bool is_k = (int)blockIdx.x >= a.q_blocks;
    const uint32_t heads = (uint32_t)(is_k ? a.k_heads : a.q_heads), per_block = 256u >> a.lane_shift, items = (uint32_t)a.T * heads;
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
    // (the same number of rounds for every thread of the block: all of them take part in the sums)
    for (uint32_t base = block * per_block; base < items; base += blocks * per_block) {
        const uint32_t item = base + (threadIdx.x >> a.lane_shift);
        const bool live = item < items && lane < a.lanes;
        const uint32_t it = live ? item : 0;
        const int token = (int)(it / heads), head = (int)(it - (uint32_t)token * heads);
        const int64_t pos = a.positions[token];
        const bool kept = pos >= 0 && pos < a.table_rows;
        const uint16_t* g = gs + token * g_row + head * g_head;
        const uint16_t* in = xs + token * x_row + head * x_head;
        const Raw<CH> g1 = load_raw<CH>(g + first), g2 = load_raw<CH>(g + second);
        Raw<CH> x1 = {}, x2 = {};
        if (weight) {
            x1 = load_raw<CH>(in + first);
            x2 = load_raw<CH>(in + second);
        }
        Angle<CH> angle;
        if (kept && turns) angle.load(a, pos, first);
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

// Values of a chunk: 8, where whole 16-byte chunks fill the rotated halves and what lies behind them.
int chunk_of(const bw_heads* h) { return h->dim % 16 == 0 && h->rotary % 16 == 0 ? 8 : 4; }

int heads_check(const bw_heads* h, int act_dtype) {
    if (!h || h->tokens < 0 || h->q_heads < 1 || h->k_heads < 1 || h->dim < 1 || h->rotary < 1 || h->rotary > h->dim || h->table_rows < 1) return BW_EINVAL;
    if (h->tokens > 0 && (!h->cos || !h->sin || !h->positions)) return BW_EINVAL;
    if (act_dtype != BW_F16 && act_dtype != BW_BF16) return BW_EUNSUPPORTED;
    if ((h->q_weight || h->k_weight) && h->weight_dtype != act_dtype && h->weight_dtype != BW_F32) return BW_EUNSUPPORTED;
    if (h->dim % 8 || h->rotary % 8 || h->dim > kMaxDim) return BW_EUNSUPPORTED;
    if (h->q_heads > 65535 || h->k_heads > 65535 || h->tokens >= (int64_t)1 << 31) return BW_EUNSUPPORTED;
    const int64_t items = h->tokens * ((int64_t)h->q_heads + h->k_heads);
    if (items >= (int64_t)1 << 31 || items * h->dim >= (int64_t)1 << 36) return BW_EUNSUPPORTED;
    if (!bw_aligned(h->cos, 16) || !bw_aligned(h->sin, 16) || !bw_aligned(h->positions, 8) || !bw_aligned(h->q_weight, 16) || !bw_aligned(h->k_weight, 16))
        return BW_EALIGN;
    return BW_OK;
}

RotateArgs args_of(const bw_heads* h) {
    RotateArgs a = {};
    a.cos = h->cos; a.sin = h->sin;
    a.positions = h->positions;
    a.q_weight = h->q_weight; a.k_weight = h->k_weight;
    a.weight_f32 = h->weight_dtype == BW_F32;
    a.table_rows = h->table_rows;
    a.T = (int)h->tokens;
    a.q_heads = h->q_heads; a.k_heads = h->k_heads;
    a.dim = h->dim;
    a.half = h->rotary / 2;
    a.lanes = h->dim / (2 * chunk_of(h));
    a.lane_shift = bw_log2(a.lanes);
    a.eps = h->eps;
    return a;
}

// Blocks of the gradient kernel for the queries or the keys: enough to fill the chip together, 1024 in proportion to their heads, so that the
// sums over them stay short (2048 tokens of 32 and 8 heads of 128, forward and backward: 30.2 us; with 768 30.5, 1536 31.9, 2048 33.1).
int grad_blocks(const bw_heads* h, int heads) {
    const int per_block = 256 >> bw_log2(h->dim / (2 * chunk_of(h))), all = h->q_heads + h->k_heads;
    const int64_t want = (h->tokens * heads + per_block - 1) / per_block, most = ((int64_t)1024 * heads + all - 1) / all;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

}  // namespace

extern "C" int bw_rotate_heads(const bw_heads* h, int act_dtype, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                               int64_t k_head, void* q_out, void* k_out, void* stream) {
    if (int st = heads_check(h, act_dtype)) return st;
    if (h->tokens == 0) return BW_OK;
    if (!q || !k || !q_out || !k_out) return BW_EINVAL;
    if (!bw_aligned(q, 16) || !bw_aligned(k, 16) || !bw_aligned(q_out, 16) || !bw_aligned(k_out, 16) || (q_row | q_head | k_row | k_head) % 8) return BW_EALIGN;
    RotateArgs a = args_of(h);
    a.q = (const uint16_t*)q; a.k = (const uint16_t*)k;
    a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head;
    a.q_out = (uint16_t*)q_out; a.k_out = (uint16_t*)k_out;
    // In several launches where a head's lanes, filled up to a power of two, would pass the 2^32 threads of one.
    const int64_t heads = h->q_heads + h->k_heads, per_block = 256 >> a.lane_shift, most = (((int64_t)1 << 32) - 256) / (heads << a.lane_shift);
    for (int64_t at = 0; at < h->tokens; at += most) {
        a.T = (int)(h->tokens - at < most ? h->tokens - at : most);
        const dim3 grid((unsigned)((a.T * heads + per_block - 1) / per_block)), block(256);
#define BW_ROTATE(DT, CH) \
    if (act_dtype == DT && chunk_of(h) == CH) hipLaunchKernelGGL((rotate_kernel<DT, CH>), grid, block, 0, (hipStream_t)stream, a);
        BW_ROTATE(BW_F16, 8) BW_ROTATE(BW_F16, 4) BW_ROTATE(BW_BF16, 8) BW_ROTATE(BW_BF16, 4)
#undef BW_ROTATE
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
        a.positions += a.T;
        a.q += a.T * q_row; a.k += a.T * k_row;
        a.q_out += (int64_t)a.T * h->q_heads * h->dim; a.k_out += (int64_t)a.T * h->k_heads * h->dim;
    }
    return BW_OK;
}

extern "C" size_t bw_rotate_heads_grad_workspace_bytes(const bw_heads* h) {
    if (heads_check(h, h && h->weight_dtype == BW_BF16 ? BW_BF16 : BW_F16) != BW_OK || (!h->q_weight && !h->k_weight)) return 0;
    return (size_t)(grad_blocks(h, h->q_heads) + grad_blocks(h, h->k_heads)) * h->dim * sizeof(float);
}

extern "C" int bw_rotate_heads_grad(const bw_heads* h, int act_dtype, const void* gq, int64_t gq_row, int64_t gq_head, const void* gk, int64_t gk_row,
                                    int64_t gk_head, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                                    void* q_grad, void* k_grad, void* q_weight_grad, void* k_weight_grad, void* workspace, size_t workspace_bytes,
                                    void* stream) {
    if (int st = heads_check(h, act_dtype)) return st;
    if ((q_weight_grad && !h->q_weight) || (k_weight_grad && !h->k_weight)) return BW_EINVAL;
    if (h->tokens > 0) {
        if (!gq || !gk || !q_grad || !k_grad || (h->q_weight && !q) || (h->k_weight && !k)) return BW_EINVAL;
        if (!bw_aligned(gq, 16) || !bw_aligned(gk, 16) || !bw_aligned(q, 16) || !bw_aligned(k, 16) || !bw_aligned(q_grad, 16) || !bw_aligned(k_grad, 16) ||
            (gq_row | gq_head | gk_row | gk_head) % 8)
            return BW_EALIGN;
        if ((h->q_weight && (q_row | q_head) % 8) || (h->k_weight && (k_row | k_head) % 8)) return BW_EALIGN;
    }
    RotateArgs a = args_of(h);
    a.gq = (const uint16_t*)gq; a.gk = (const uint16_t*)gk;
    a.gq_row = gq_row; a.gq_head = gq_head; a.gk_row = gk_row; a.gk_head = gk_head;
    a.q = (const uint16_t*)q; a.k = (const uint16_t*)k;
    a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head;
    a.q_out = (uint16_t*)q_grad; a.k_out = (uint16_t*)k_grad;
    a.q_blocks = h->tokens ? grad_blocks(h, h->q_heads) : 0;
    const int blocks = h->tokens ? a.q_blocks + grad_blocks(h, h->k_heads) : 0;
    const bool sums = q_weight_grad || k_weight_grad;
    if (sums && blocks) {
        if (!workspace || workspace_bytes < bw_rotate_heads_grad_workspace_bytes(h)) return BW_EWORKSPACE;
        if (!bw_aligned(workspace, 16)) return BW_EALIGN;
        a.partial = (float*)workspace;
    }
    if (blocks) {
#define BW_ROTATE(DT, CH) \
    if (act_dtype == DT && chunk_of(h) == CH) hipLaunchKernelGGL((rotate_grad_kernel<DT, CH>), dim3(blocks), dim3(256), 0, (hipStream_t)stream, a);
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
