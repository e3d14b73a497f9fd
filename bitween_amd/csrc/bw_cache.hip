// Writing tokens into the paged key-value cache, quantised as they are written, and reading them back.
//
// A thread owns 8 or 16 consecutive values of one token's key or value head.  The 2 ... 8 neighbouring threads of a group agree on its extrema with
// cross-lane moves (their number divides 64 and every row starts at a multiple of it, so a group never leaves its wave), and the first of
// them stores the group's pair.
//
// The code of x is rint(x / s) of the exact quotient: with r = 1 / s to within a unit of its last place, t = x r and one step t + (x - t s) r the
// result is the correctly rounded quotient wherever rint could tell a difference - x has at most 11 significant bits and s 11, so a
// quotient up to 256 that is not exactly half way between two whole numbers lies at least 2^-13 from half way, and one that is half way has at
// most 10 bits, which the step returns exactly (the residual is exact in the fused operation).  The range over 15 or 255 is that step too, with the
// correctly rounded reciprocal: the correctly rounded quotient (checked over a whole binade and samples of all others).
//
// Extrema of 16-bit floats are whole-number maxima of their bits: a positive value's bits grow with it, a negative one's are negative, so
// max(0, bits) over a group is its largest value (or 0), max(0, bits ^ sign) its most negative one, and an infinity or a NaN shows as bits from the
// infinity's on.  Both fit one register on the way over the lanes.
//
// Both kernels are one pass over memory: what bounds them is HBM beyond a few hundred tokens and the launch below.  32768 tokens of 8 heads of 128
// at 8 bits (203 MB each way): 38 us to write, 36 us to read back, 5.3 and 5.6 TB/s; a copy reaches 5.2.
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
    int T, heads, groups, dim;
    FastDiv units, chunks;                       // threads of a token (2 * heads * chunks) and of a head
    int page_shift, group_shift;                 // 1 << group_shift threads for a group
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
    uint32_t at, chunk;
    u.token = (int)a.units.div(i, at);
    const uint32_t head = a.chunks.div(at, chunk);             // keys' heads, then values'
    u.value = head >= (uint32_t)a.heads;
    u.head = (int)head - (u.value ? a.heads : 0);
    u.chunk = (int)chunk;
    return u;
}

// Larger of the two 16-bit whole numbers of each half.
typedef short s2 __attribute__((ext_vector_type(2)));
BW_DEV uint32_t max16(uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s2, a), __builtin_bit_cast(s2, b))); }
template <int CTRL> BW_DEV uint32_t max16_over(uint32_t v) { return max16(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false)); }

// Workgroups go to the eight dies in turn: here each die gets kRun neighbouring ones of every 8 kRun, so that the pairs of neighbouring tokens,
// which share lines, are put together in one die's cache.
constexpr uint32_t kRun = 32;
BW_DEV uint32_t block_of(uint32_t b, uint32_t n) {
    const uint32_t at = b & (8 * kRun - 1), base = b - at;
    return base + 8 * kRun <= n ? base + (at & 7) * kRun + (at >> 3) : b;
}

// Values of a thread: for codes 16, so that the two thirds of the work that are a group's and an address's are shared by more of them (with 8: 49 us
// for the case below, 380 operations for 16 values against 230).
template <int BITS> constexpr int kWriteValues = BITS == 16 ? 8 : 16;

template <int DT, int BITS>
__global__ __launch_bounds__(256) void cache_write_kernel(CacheArgs a) {
    constexpr int V = kWriteValues<BITS>;
    const uint32_t i = block_of(blockIdx.x, gridDim.x) * 256u + threadIdx.x;
    const bool live = i < (uint32_t)a.T * a.units.d;
    const Unit u = unit_of(a, live ? i : 0);
    const int64_t slot = a.slots[u.token];
    const bool kept = live && slot >= 0 && slot < a.rows;
    const uint16_t* src = (u.value ? a.v + u.token * a.v_row + u.head * a.v_head : a.k + u.token * a.k_row + u.head * a.k_head) + u.chunk * V;
    uint32_t w[V / 2];
#pragma unroll
    for (int n = 0; n < V / 8; n++) {
        const u4 t = reinterpret_cast<const u4*>(src)[n];
#pragma unroll
        for (int j = 0; j < 4; j++) w[4 * n + j] = t[j];
    }
    uint8_t* out = u.value ? a.values : a.keys;
    if constexpr (BITS == 16) {
        if (kept) *reinterpret_cast<u4*>(out + (row_index(a, slot, u.head) * a.dim + u.chunk * 8) * 2) = u4{w[0], w[1], w[2], w[3]};
    } else {
        constexpr float top = (float)((1 << BITS) - 1), inv_top = 1.f / top;
        uint32_t hi = 0, lo = 0;
#pragma unroll
        for (int j = 0; j < V / 2; j++) {
            hi = max16(hi, w[j]);
            lo = max16(lo, w[j] ^ 0x80008000u);
        }
        // low half: the largest value, high half: the size of the most negative one
        uint32_t both = max16(__builtin_amdgcn_perm(lo, hi, 0x05040100u), __builtin_amdgcn_perm(lo, hi, 0x07060302u));
        both = max16_over<0xB1>(both);                          // quad_perm: the neighbour
        if (a.group_shift > 1) both = max16_over<0x4E>(both);   // ... and the other two of four
        if (a.group_shift > 2) both = max16_over<0x141>(both);  // row_half_mirror: the other four of eight
        constexpr uint32_t inf = DT == BW_F16 ? 0x7C00u : 0x7F80u;
        const bool bad = (both & 0xFFFFu) >= inf || (both >> 16) >= inf;
        const float largest = widen16<DT>((uint16_t)both), smallest = -widen16<DT>((uint16_t)(both >> 16));
        // the scale rounds up, so that no code has to be clipped for its rounding; never 0
        const float range = largest - smallest, t0 = range * inv_top;
        const float step = fminf(__builtin_fmaf(__builtin_fmaf(-t0, top, range), inv_top, t0), 65504.f);
        uint32_t sb = __builtin_bit_cast(uint16_t, (_Float16)step);
        sb += f16_bits(sb) < step ? 1 : 0;
        sb = sb ? sb : 1;
        const float s = f16_bits(sb), r = __builtin_amdgcn_rcpf(s);
        // 1.5 2^23 added: the nearest whole number (ties to even) in the low bits, and whole numbers may be added to it
        constexpr float kWhole = 12582912.f;
        auto whole = [&](float v) {
            const float t = v * r;
            return __builtin_fmaf(__builtin_fmaf(-t, s, v), r, t) + kWhole;
        };
        const float z = fminf(whole(-smallest) - kWhole, top);
        uint32_t q[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float x = whole(widen16<DT>((uint16_t)(w[j / 2] >> (16 * (j & 1))))) + z;
            q[j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_fmed3f(x, kWhole, kWhole + top));   // (a group with a NaN is marked by its scale)
        }
        if (kept) {
            auto bytes = [](uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
                return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b3, b2, 0x0C0C0400u), __builtin_amdgcn_perm(b1, b0, 0x0C0C0400u), 0x05040100u);
            };
            uint8_t* dst = out + row_index(a, slot, u.head) * (a.dim * BITS / 8) + u.chunk * (V * BITS / 8);
            if constexpr (BITS == 8) {
                *reinterpret_cast<u4*>(dst) = u4{bytes(q[0], q[1], q[2], q[3]), bytes(q[4], q[5], q[6], q[7]), bytes(q[8], q[9], q[10], q[11]), bytes(q[12], q[13], q[14], q[15])};
            } else {
                *reinterpret_cast<u2*>(dst) = u2{bytes(q[0] | q[1] << 4, q[2] | q[3] << 4, q[4] | q[5] << 4, q[6] | q[7] << 4),
                                                 bytes(q[8] | q[9] << 4, q[10] | q[11] << 4, q[12] | q[13] << 4, q[14] | q[15] << 4)};
            }
            if ((u.chunk & ((1 << a.group_shift) - 1)) == 0)
                (u.value ? a.value_meta : a.key_meta)[pair_index(a, slot, u.head, u.chunk >> a.group_shift)] =
                    (bad ? 0x7E00u : sb) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)z) << 16;
        }
    }
}

template <int DT, int BITS>
BW_DEV u4 read_unit(const CacheArgs& a, const Unit& u, int64_t slot) {
    const uint8_t* in = u.value ? a.values : a.keys;
    u4 w = {0, 0, 0, 0};
    if (slot >= 0 && slot < a.rows) {
        if constexpr (BITS == 16) {
            w = *reinterpret_cast<const u4*>(in + (row_index(a, slot, u.head) * a.dim + u.chunk * 8) * 2);
        } else {
            const uint8_t* src = in + row_index(a, slot, u.head) * (a.dim * BITS / 8) + u.chunk * BITS;
            const uint32_t pair = (u.value ? a.value_meta : a.key_meta)[pair_index(a, slot, u.head, u.chunk >> a.group_shift)];
            uint32_t words[BITS / 4];
            if constexpr (BITS == 8) { const u2 t = *reinterpret_cast<const u2*>(src); words[0] = t[0]; words[1] = t[1]; }
            else words[0] = *reinterpret_cast<const uint32_t*>(src);
            h2 v[4];                                             // q - z, exact
            GroupConstNat<BITS> g;
            g.set(as_h2(pair)[0], as_h2(pair)[1]);
            if constexpr (BITS == 8) {
                dequant_word8_nat<false>(words[0], g, v);
                dequant_word8_nat<false>(words[1], g, v + 2);
            } else {
                dequant_word4_nat<false>(words[0], g, v);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (DT == BW_F16) {                    // one rounding; beyond the largest number: that number; a NaN scale: NaN
                    const h2 most = splat((_Float16)65504.f);
                    w[j] = as_u32(__builtin_elementwise_max(__builtin_elementwise_min(v[j] * g.s, most), -most) + (g.s - g.s));
                } else {
                    w[j] = narrow_pair<DT>((float)v[j][0] * (float)g.s[0], (float)v[j][1] * (float)g.s[0]);
                }
            }
        }
    }
    return w;
}

// UN chunks of a thread, 256 chunks apart, all under way at a time.
template <int DT, int BITS, int UN>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheArgs a) {
    const uint32_t first = block_of(blockIdx.x, gridDim.x) * (256u * UN) + threadIdx.x, all = (uint32_t)a.T * a.units.d;
    Unit u[UN];
    int64_t slot[UN];
    u4 w[UN];
#pragma unroll
    for (int n = 0; n < UN; n++) {
        const uint32_t i = first + 256 * n;
        u[n] = unit_of(a, i < all ? i : 0);
        slot[n] = a.slots[u[n].token];
    }
#pragma unroll
    for (int n = 0; n < UN; n++) w[n] = read_unit<DT, BITS>(a, u[n], slot[n]);
#pragma unroll
    for (int n = 0; n < UN; n++) {
        uint16_t* out = (u[n].value ? a.v_out : a.k_out) + ((int64_t)u[n].token * a.heads + u[n].head) * a.dim + u[n].chunk * 8;
        if (first + 256 * n >= all) continue;
        if constexpr (UN > 1) __builtin_nontemporal_store(w[n], reinterpret_cast<u4*>(out));
        else *reinterpret_cast<u4*>(out) = w[n];
    }
}

// Two pieces of memory of `bytes` that share some.
bool overlap(const void* a, const void* b, int64_t bytes) {
    const int64_t apart = (int64_t)((const char*)a - (const char*)b);
    return apart < bytes && apart > -bytes;
}

CacheArgs args_of(const bw_cache* c, int values) {
    CacheArgs a{};
    a.keys = (uint8_t*)c->keys;
    a.values = (uint8_t*)c->values;
    a.key_meta = (uint32_t*)c->key_meta;
    a.value_meta = (uint32_t*)c->value_meta;
    a.rows = c->pages * c->page_size;
    a.heads = c->kv_heads;
    a.dim = c->dim;
    a.chunks = FastDiv(c->dim / values);
    a.units = FastDiv(2 * c->kv_heads * (c->dim / values));
    a.page_shift = bw_log2(c->page_size);
    if (c->bits != 16) {
        a.groups = c->dim / c->group;
        a.group_shift = bw_log2(c->group / values);
    }
    return a;
}

// Chunks (of 16 bytes) from which on a thread of the read-back takes kAhead of them (36 -> 33 us for the case above; four: no further) and stores
// past the caches: 17 MB and more leave no room for what else a step reads (12289 tokens of 12 heads of 64 at 4 bits 11.3 -> 9.8 us; written
// and read back in turns, the case above 79 -> 74 us).
constexpr int kAhead = 2;
constexpr int64_t kManyChunks = (int64_t)kAhead * 256 * 2048;

// Runs `launch(args, chunks)` over the tokens, in several launches where a thread's number would pass 31 bits.
template <class F>
int over_tokens(CacheArgs a, int64_t T, F&& launch) {
    const int64_t most = ((int64_t)1 << 31) / a.units.d - 1;
    for (int64_t at = 0; at < T; at += most) {
        CacheArgs b = a;
        b.T = (int)(T - at < most ? T - at : most);
        b.slots += at;
        if (b.k) { b.k += at * a.k_row; b.v += at * a.v_row; }
        if (b.k_out) { b.k_out += at * a.heads * a.dim; b.v_out += at * a.heads * a.dim; }
        launch(b, (int64_t)b.T * a.units.d);
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    return BW_OK;
}

template <int DT, int BITS> void launch_write(const CacheArgs& a, int64_t chunks, hipStream_t stream) {
    hipLaunchKernelGGL((cache_write_kernel<DT, BITS>), dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, stream, a);
}
template <int DT, int BITS> void launch_read(const CacheArgs& a, int64_t chunks, hipStream_t stream) {
    if (chunks < kManyChunks) hipLaunchKernelGGL((cache_read_kernel<DT, BITS, 1>), dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((cache_read_kernel<DT, BITS, kAhead>), dim3((unsigned)((chunks + 256 * kAhead - 1) / (256 * kAhead))), dim3(256), 0, stream, a);
}

}  // namespace

#define BW_BY_FORMAT(LAUNCH, DT)                                       \
    over_tokens(a, T, [&](const CacheArgs& b, int64_t chunks) {        \
        if (c->bits == 16) LAUNCH<DT, 16>(b, chunks, (hipStream_t)stream);     \
        else if (c->bits == 8) LAUNCH<DT, 8>(b, chunks, (hipStream_t)stream);  \
        else LAUNCH<DT, 4>(b, chunks, (hipStream_t)stream);            \
    })

extern "C" int bw_cache_write(const bw_cache* c, int act_dtype, int64_t T, const void* k, int64_t k_row, int64_t k_head, const void* v,
                              int64_t v_row, int64_t v_head, const int64_t* slots, void* stream) {
    if (int st = bw_cache_check(c)) return st;
    if (T < 0 || (T > 0 && (!k || !v || !slots))) return BW_EINVAL;
    if ((act_dtype != BW_F16 && act_dtype != BW_BF16) || (c->bits == 16 && act_dtype != c->dtype)) return BW_EUNSUPPORTED;
    if (T == 0) return BW_OK;
    if (!bw_aligned(k, 16) || !bw_aligned(v, 16) || !bw_aligned(slots, 8) || (k_row | k_head | v_row | v_head) % 8) return BW_EALIGN;
    const int64_t values = c->pages * c->page_size * c->kv_heads * c->dim;
    if (overlap(c->keys, c->values, values / 8 * c->bits) || (c->bits != 16 && overlap(c->key_meta, c->value_meta, values / c->group * 4))) return BW_EINVAL;
    CacheArgs a = args_of(c, c->bits == 16 ? kWriteValues<16> : kWriteValues<8>);
    a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
    a.k_row = k_row; a.k_head = k_head; a.v_row = v_row; a.v_head = v_head;
    a.slots = slots;
    return act_dtype == BW_F16 ? BW_BY_FORMAT(launch_write, BW_F16) : BW_BY_FORMAT(launch_write, BW_BF16);
}

extern "C" int bw_cache_read(const bw_cache* c, int out_dtype, int64_t T, const int64_t* slots, void* k_out, void* v_out, void* stream) {
    if (int st = bw_cache_check(c)) return st;
    if (T < 0 || (T > 0 && (!slots || !k_out || !v_out))) return BW_EINVAL;
    if ((out_dtype != BW_F16 && out_dtype != BW_BF16) || (c->bits == 16 && out_dtype != c->dtype)) return BW_EUNSUPPORTED;
    if (T == 0) return BW_OK;
    if (!bw_aligned(k_out, 16) || !bw_aligned(v_out, 16) || !bw_aligned(slots, 8)) return BW_EALIGN;
    CacheArgs a = args_of(c, 8);
    a.slots = slots;
    a.k_out = (uint16_t*)k_out; a.v_out = (uint16_t*)v_out;
    return out_dtype == BW_F16 ? BW_BY_FORMAT(launch_read, BW_F16) : BW_BY_FORMAT(launch_read, BW_BF16);
}
