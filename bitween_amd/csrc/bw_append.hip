// Queries, keys and values of new tokens in one launch: queries and keys rotated (bw_rotate.h has which values a thread owns), keys and values into their
// rows of the paged cache, quantised on the way (bw_cache.h).
//
// A head's threads hold chunks of CH values from both halves of the rotation, so the threads of a group of values to quantise are not neighbours in general: every
// thread leaves its chunks' extrema in LDS, where a head's chunks lie in order, and reads those of its groups; a head never leaves its wave, so that nothing
// waits but the wave.
//
// One pass over memory: launch-bound up to a few hundred tokens (one token 2.4 us; 64 with norms into 8 bits 4.7), HBM beyond: 8191 tokens of 32 and 8 heads of 128 by three axes into 4 bits
// 38 us (177 MB, 4.7 TB/s; 59 with one head to a thread, which loads its angles from three rows of the tables for each).
//
// The codes hang on the rotated key's last bit next to a border, so what goes into it is kept reproducible: the sum of squares and its root are float64
// (whose order no longer shows), the rest are single float32 operations.  64-bit operations cost what 32-bit ones do here, twice over, and memory is waited for either way.
#include "bw_rotate.h"

namespace {

struct AppendArgs {
    const uint16_t* v;
    int64_t v_row, v_head;
    const int64_t* slots;
    uint8_t *keys, *values;
    uint32_t *key_meta, *value_meta;
    int64_t rows;                                // of the cache: pages * page_size
    int kv_heads, groups, page_shift, group_chunks;      // chunks of CH values of a group
};

template <int DT> BW_DEV double wide_sum(double v, int shift) {
    auto add = [&](auto&& other) {
        const uint64_t bits = __builtin_bit_cast(uint64_t, v);
        const float lo = other(__builtin_bit_cast(float, (uint32_t)bits)), hi = other(__builtin_bit_cast(float, (uint32_t)(bits >> 32)));
        v += __builtin_bit_cast(double, (uint64_t)__builtin_bit_cast(uint32_t, hi) << 32 | __builtin_bit_cast(uint32_t, lo));
    };
    if (shift > 0) add([](float x) { return from_lane<0xB1>(x); });
    if (shift > 1) add([](float x) { return from_lane<0x4E>(x); });
    if (shift > 2) add([](float x) { return from_lane<0x141>(x); });
    if (shift > 3) add([](float x) { return from_lane<0x140>(x); });
    if (shift > 4) add([](float x) { return __shfl_xor(x, 16, 64); });
    return v;
}
// 1 / sqrt(x), to within a few units of a float64's last place: two steps from the instruction's 2^-14 or better.  Of an infinity 0, which the steps would make NaN: what is
// finite in such a head is 0 then.
BW_DEV double rsqrt_wide(double x) {
    double y = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; i++) y = __builtin_fma(y, 0.5 * __builtin_fma(-x * y, y, 1.0), y);
    return x == __builtin_inf() ? 0.0 : y;
}

// A thread has its place in some of a token's heads, a.slices apart: the queries', the keys' and the values', and their angles once.
template <int DT, int CH, bool AXES, int BITS>
__global__ __launch_bounds__(256) void append_kernel(RotateArgs a, AppendArgs c) {
    __shared__ __align__(16) uint32_t extrema[BITS == 16 ? 4 : 512];
    const uint32_t units = (uint32_t)(a.q_heads + 2 * c.kv_heads), item = (blockIdx.x * 256 + threadIdx.x) >> a.lane_shift;
    const int lane = (int)threadIdx.x & ((1 << a.lane_shift) - 1);
    const bool there = item < (uint32_t)a.T * a.slices, live = there && lane < a.lanes;
    const uint32_t it = there ? item : 0;                        // (lanes that fill a head up are of its kind)
    const int token = (int)(it / a.slices);
    int first, second;
    bool turns;
    chunks_of<CH>(a, live ? lane : 0, first, second, turns);
    auto source = [&](int unit) {
        return unit < a.q_heads ? a.q + token * a.q_row + unit * a.q_head : unit < a.q_heads + c.kv_heads ? a.k + token * a.k_row + (unit - a.q_heads) * a.k_head
                                                                          : c.v + token * c.v_row + (unit - a.q_heads - c.kv_heads) * c.v_head;
    };
    uint32_t unit = it - (uint32_t)token * a.slices;
    const uint16_t* src = source((int)unit);
    Raw<CH> raw[2] = {load_raw<CH>(src + first), load_raw<CH>(src + second)};
    const int64_t slot = c.slots[token];
    const Position<AXES> pos(a, token);
    Angle<CH> angle;
    if (pos.kept && turns && unit < (uint32_t)(a.q_heads + c.kv_heads)) angle.load(a, pos, first);
    const bool kept = live && pos.kept && slot >= 0 && slot < c.rows;
    const int64_t page = slot >> c.page_shift, in_page = slot & ((1 << c.page_shift) - 1);
    auto store = [](void* p, const uint32_t* w) {
        if constexpr (CH == 8) *reinterpret_cast<u4*>(p) = u4{w[0], w[1], w[2], w[3]};
        else *reinterpret_cast<u2*>(p) = u2{w[0], w[1]};
    };
    for (;;) {
        const uint32_t next = unit + a.slices;
        const bool more = next < units, is_q = unit < (uint32_t)a.q_heads, is_v = unit >= (uint32_t)(a.q_heads + c.kv_heads), is_k = !is_q && !is_v;
        const int head = (int)unit - (is_q ? 0 : is_v ? a.q_heads + c.kv_heads : a.q_heads);
        src = source((int)(more ? next : unit));
        const Raw<CH> after[2] = {load_raw<CH>(src + first), load_raw<CH>(src + second)};
        uint32_t w[2][CH / 2];                                   // the chunks as they are stored
#pragma unroll
        for (int j = 0; j < CH / 2; j++) { w[0][j] = raw[0][j]; w[1][j] = raw[1][j]; }
        if (!is_v) {
            float x[CH], y[CH];
            widen_raw<DT, CH>(raw[0], x);
            widen_raw<DT, CH>(raw[1], y);
            const void* weight = is_k ? a.k_weight : a.q_weight;
            if (weight) {
                double ss = 0.;
                if (live) {
#pragma unroll
                    for (int j = 0; j < CH; j++) ss = __builtin_fma((double)x[j], (double)x[j], __builtin_fma((double)y[j], (double)y[j], ss));
                }
                const float r = (float)rsqrt_wide(wide_sum<DT>(ss, a.lane_shift) / a.dim + (double)a.eps);
                float g[CH];
                load_weight<DT, CH>(weight, a.weight_f32, first, g);
#pragma unroll
                for (int j = 0; j < CH; j++) x[j] = x[j] * r * g[j];
                load_weight<DT, CH>(weight, a.weight_f32, second, g);
#pragma unroll
                for (int j = 0; j < CH; j++) y[j] = y[j] * r * g[j];
            }
            if (pos.kept && turns) angle.template turn<1>(x, y);
#pragma unroll
            for (int j = 0; j < CH / 2; j++) {
                w[0][j] = narrow_pair<DT>(x[2 * j], x[2 * j + 1]);
                w[1][j] = narrow_pair<DT>(y[2 * j], y[2 * j + 1]);
            }
        }
        const int64_t row = ((page * c.kv_heads + head) << c.page_shift) + in_page;
        uint8_t* out = is_v ? c.values : c.keys;
        if (is_q) {
            if (live) {
                uint16_t* to = a.q_out + ((int64_t)token * a.q_heads + head) * a.dim;
                if (!pos.kept) {
#pragma unroll
                    for (int j = 0; j < CH / 2; j++) w[0][j] = w[1][j] = 0;
                }
                store(to + first, w[0]);
                store(to + second, w[1]);
            }
        } else if constexpr (BITS == 16) {
            if (kept) {
                store(out + (row * a.dim + first) * 2, w[0]);
                store(out + (row * a.dim + second) * 2, w[1]);
            }
        } else {
            // (a head's lanes are all here; those of queries leave nothing in LDS)
            uint32_t* mine = extrema + ((threadIdx.x >> 6) * 128 + ((threadIdx.x & 63) >> a.lane_shift << (a.lane_shift + 1)));
            if (lane < a.lanes) {
                mine[first / CH] = extrema_of<CH / 2>(w[0]);
                mine[second / CH] = extrema_of<CH / 2>(w[1]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            uint32_t* meta = is_v ? c.value_meta : c.key_meta;
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int at = n ? second : first, chunk = at / CH, group = chunk / c.group_chunks;
                const u4* from = reinterpret_cast<const u4*>(mine + group * c.group_chunks);
                uint32_t both = 0;
                if (lane < a.lanes) {
                    for (int i = 0; i < c.group_chunks / 4; i++) {
                        const u4 t = from[i];
                        both = max16(both, max16(max16(t[0], t[1]), max16(t[2], t[3])));
                    }
                }
                const GroupCoder<DT, BITS> coder(both);
                uint32_t q[CH];
#pragma unroll
                for (int j = 0; j < CH; j++) q[j] = coder.code(widen16<DT>((uint16_t)(w[n][j / 2] >> (16 * (j & 1)))));
                if (!kept) continue;
                uint8_t* dst = out + row * (a.dim * BITS / 8) + at * BITS / 8;
                if constexpr (BITS == 8 && CH == 8) *reinterpret_cast<u2*>(dst) = u2{bytes_of(q[0], q[1], q[2], q[3]), bytes_of(q[4], q[5], q[6], q[7])};
                else if constexpr (BITS == 8) *reinterpret_cast<uint32_t*>(dst) = bytes_of(q[0], q[1], q[2], q[3]);
                else if constexpr (CH == 8) *reinterpret_cast<uint32_t*>(dst) = bytes_of(q[0] | q[1] << 4, q[2] | q[3] << 4, q[4] | q[5] << 4, q[6] | q[7] << 4);
                else *reinterpret_cast<uint16_t*>(dst) = (uint16_t)bytes_of(q[0] | q[1] << 4, q[2] | q[3] << 4, 0, 0);
                if (chunk % c.group_chunks == 0) meta[(((page * c.kv_heads + head) * c.groups + group) << c.page_shift) + in_page] = coder.pair;
            }
            // (the next head's extrema go where these are read)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        if (!more) return;
        unit = next;
        raw[0] = after[0];
        raw[1] = after[1];
    }
}

template <int DT, int CH, bool AXES>
void launch_append(const RotateArgs& a, const AppendArgs& c, int bits, dim3 grid, hipStream_t stream) {
    if (bits == 16) hipLaunchKernelGGL((append_kernel<DT, CH, AXES, 16>), grid, dim3(256), 0, stream, a, c);
    else if (bits == 8) hipLaunchKernelGGL((append_kernel<DT, CH, AXES, 8>), grid, dim3(256), 0, stream, a, c);
    else hipLaunchKernelGGL((append_kernel<DT, CH, AXES, 4>), grid, dim3(256), 0, stream, a, c);
}

}  // namespace

extern "C" int bw_cache_append(const bw_cache* cache, const bw_heads* h, const bw_axes* axes, int act_dtype, const void* q, int64_t q_row, int64_t q_head,
                               const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const int64_t* slots, void* q_out,
                               void* stream) {
    if (int st = bw_cache_check(cache)) return st;
    if (int st = heads_check(h, act_dtype)) return st;
    if (axes)
        if (int st = axes_check(axes, h->rotary)) return st;
    if (h->k_heads != cache->kv_heads || h->dim != cache->dim) return BW_EINVAL;
    if (cache->bits == 16 && act_dtype != cache->dtype) return BW_EUNSUPPORTED;
    const int64_t units = h->q_heads + 2 * (int64_t)h->k_heads;
    if (h->tokens * units >= (int64_t)1 << 31) return BW_EUNSUPPORTED;
    if (h->tokens == 0) return BW_OK;
    if (!q || !k || !v || !slots || !q_out) return BW_EINVAL;
    if (!bw_aligned(q, 16) || !bw_aligned(k, 16) || !bw_aligned(v, 16) || !bw_aligned(q_out, 16) || !bw_aligned(slots, 8) ||
        (q_row | q_head | k_row | k_head | v_row | v_head) % 8)
        return BW_EALIGN;
    const int64_t values = cache->pages * cache->page_size * cache->kv_heads * cache->dim;
    if (bw_overlap(cache->keys, cache->values, values / 8 * cache->bits) || (cache->bits != 16 && bw_overlap(cache->key_meta, cache->value_meta, values / cache->group * 4)))
        return BW_EINVAL;
    RotateArgs a = rotate_args(h, axes);
    a.q = (const uint16_t*)q; a.k = (const uint16_t*)k;
    a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head;
    a.q_out = (uint16_t*)q_out;
    AppendArgs c = {};
    c.v = (const uint16_t*)v; c.v_row = v_row; c.v_head = v_head;
    c.slots = slots;
    c.keys = (uint8_t*)cache->keys; c.values = (uint8_t*)cache->values;
    c.key_meta = (uint32_t*)cache->key_meta; c.value_meta = (uint32_t*)cache->value_meta;
    c.rows = cache->pages * cache->page_size;
    c.kv_heads = cache->kv_heads;
    c.page_shift = bw_log2(cache->page_size);
    const int chunk = chunk_of(h);
    if (cache->bits != 16) {
        c.groups = cache->dim / cache->group;
        c.group_chunks = cache->group / chunk;
    }
    // In several launches where a head's lanes, filled up to a power of two, would pass the 2^32 threads of one.
    const int64_t per_block = 256 >> a.lane_shift, most = (((int64_t)1 << 32) - 256) / (units << a.lane_shift);
    for (int64_t at = 0; at < h->tokens; at += most) {
        a.T = (int)(h->tokens - at < most ? h->tokens - at : most);
        a.slices = (uint32_t)slices_of(a, (int)units);
        const dim3 grid((unsigned)(((int64_t)a.T * a.slices + per_block - 1) / per_block));
#define BW_APPEND(DT, CH) \
    if (act_dtype == DT && chunk == CH && axes) launch_append<DT, CH, true>(a, c, cache->bits, grid, (hipStream_t)stream); \
    else if (act_dtype == DT && chunk == CH) launch_append<DT, CH, false>(a, c, cache->bits, grid, (hipStream_t)stream);
        BW_APPEND(BW_F16, 8) BW_APPEND(BW_F16, 4) BW_APPEND(BW_BF16, 8) BW_APPEND(BW_BF16, 4)
#undef BW_APPEND
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
        a.positions += a.T;
        a.q += a.T * q_row; a.k += a.T * k_row; c.v += a.T * v_row;
        c.slots += a.T;
        a.q_out += (int64_t)a.T * h->q_heads * h->dim;
    }
    return BW_OK;
}
