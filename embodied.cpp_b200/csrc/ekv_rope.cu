// ekv_rope.cu -- rotary positions on q and k, with the rotated k and the v written into the pool's pages.
//
// Pair i of a head turns by pos * f_i: (a, b) -> mag * (a cos - b sin, a sin + b cos). The angle is taken in
// turns, pos * (f_i / 2 pi) in 64 bits, reduced to its fraction, and only then rounded to 32: at position
// 100000 a 32-bit product would be off by 0.004 radians. One CTA computes the sines of its rows once and uses
// them for every head; the rest is a stream of 16-byte loads and stores.
// Bound: DRAM. On the device 32 k rows of 48 heads of 128 columns (700 MB read and written) take 118 us, 5.9 TB/s, 91% of the
// measured copy rate (125 us, 85%, as calls with inputs that change); 3 k rows of 10 heads of 256 (31 MB) 9.1 us, half of it
// the dependent loads before the stream (rows of the request, their positions, the sines); one row 3.7 us. 8-bit pages are
// written a 32-column group a thread, read column by column: 233 us for the 32 k rows' like, whose bytes take 113.
#include <algorithm>
#include <cmath>
#include <new>

#include "ekv_decode.cuh"
#include "ekv_internal.h"

struct ekv_rope {
    int32_t device, interleaved, rotary;
    float magnitude;
    double freq[128];      // radians per position of each pair
    double *dev_turns;     // the same in turns, on the device
};

namespace ekv {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRows = 8;  // rows per CTA
constexpr int kLoads = 2;    // units (of 16 or 32 bytes) a thread loads before it stores

// Division of small numbers by a fixed one: floor(i / d) = (i * ceil(2^32 / d)) >> 32 while i * d < 2^32.
struct SmallDiv {
    uint32_t m;
    SmallDiv() = default;
    explicit SmallDiv(uint32_t d) : m((uint32_t)(((1ull << 32) + d - 1) / d)), one(d == 1) {}
    uint32_t one;
    __device__ __forceinline__ int operator()(int i) const { return one ? i : (int)__umulhi((uint32_t)i, m); }
};

struct RopeArgs {
    PoolView pool;
    int32_t layer, n_batch, max_rows, rows_per_cta, q_heads, interleaved, rotary;
    int32_t per;       // units of a turned head
    int32_t per_item;  // items of a query head that is turned in place in the odd form, else 0
    SmallDiv div_per, div_item, div_q, div_kv, div_v;
    float magnitude;
    const double *turns;
    const int32_t *seq_ids, *dst_pos, *n_rows, *src_row, *positions;
    const uint16_t *q, *k, *v;
    int64_t q_stride, kv_stride;  // elements per source row
    uint16_t *q_out;
};

// An interleaved pair in one word. Which product is rounded and which is part of the sum is said, so that every form gives
// the same bits: left to the compiler it differed from form to form, and two of 10^7 values with it.
__device__ __forceinline__ uint32_t rot_pair(uint32_t lo_hi, float2 cs) {
    const float x = bf16_bits_to_f32((uint16_t)lo_hi), y = bf16_bits_to_f32((uint16_t)(lo_hi >> 16));
    const uint32_t a = f32_to_bf16_bits(__fmaf_rn(x, cs.x, -__fmul_rn(y, cs.y))), b = f32_to_bf16_bits(__fmaf_rn(x, cs.y, __fmul_rn(y, cs.x)));
    return a | b << 16;
}

// One head's unit u: 16 bytes, or the two 16-byte halves of eight split pairs (the columns past the rotated ones
// follow them, 16 bytes each).
struct Unit {
    uint4 x, y;
};
__device__ __forceinline__ Unit load_unit(const RopeArgs &a, const uint16_t *src, int u) {
    Unit r;
    const int n = a.rotary, pairs = n / 16;
    const bool pair = !a.interleaved && u < pairs;
    const int d = a.interleaved || pair ? 8 * u : n + 8 * (u - pairs);
    r.x = *(const uint4 *)(src + d);
    r.y = pair ? *(const uint4 *)(src + d + n / 2) : make_uint4(0, 0, 0, 0);
    return r;
}
// `put(d, value)` writes the 16 bytes of columns d .. d + 7.
template <class Put>
__device__ __forceinline__ void turn_unit(const RopeArgs &a, Unit r, int u, const float2 *cs, Put put) {
    const int n = a.rotary;
    if (a.interleaved) {
        const int d = 8 * u;
        if (d < n) {
            r.x.x = rot_pair(r.x.x, cs[d / 2]);
            if (d + 2 < n) r.x.y = rot_pair(r.x.y, cs[d / 2 + 1]);
            if (d + 4 < n) r.x.z = rot_pair(r.x.z, cs[d / 2 + 2]);
            if (d + 6 < n) r.x.w = rot_pair(r.x.w, cs[d / 2 + 3]);
        }
        put(d, r.x);
        return;
    }
    const int pairs = n / 16;
    if (u >= pairs) {
        put(n + 8 * (u - pairs), r.x);
        return;
    }
    const int d = 8 * u, h = n / 2;
    const uint32_t xs[4] = {r.x.x, r.x.y, r.x.z, r.x.w}, ys[4] = {r.y.x, r.y.y, r.y.z, r.y.w};
    uint32_t p[4], q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 c = *(const float4 *)&cs[d + 2 * i];
        const uint32_t e = rot_pair((xs[i] & 0xffffu) | ys[i] << 16, make_float2(c.x, c.y));
        const uint32_t o = rot_pair(xs[i] >> 16 | (ys[i] & 0xffff0000u), make_float2(c.z, c.w));
        p[i] = (e & 0xffffu) | o << 16;
        q[i] = e >> 16 | (o & 0xffff0000u);
    }
    put(d, make_uint4(p[0], p[1], p[2], p[3]));
    put(d + h, make_uint4(q[0], q[1], q[2], q[3]));
}

// The odd form: split pairs that are not whole 16-byte units. Columns 8 u .. 8 u + 7 of the result, whose partners are
// read one by one: 9 of 32 units where 66 of 256 columns turn (8 x 2000 rows of 16 such heads and v: 222 -> 131 us against
// pair by pair; 64 columns, in whole units: 73).
__device__ __forceinline__ uint4 odd_unit(const RopeArgs &a, const uint16_t *src, int u, const float2 *cs) {
    const uint4 own = *(const uint4 *)(src + 8 * u);
    const int n = a.rotary, h = n / 2;
    if (8 * u >= n) return own;
    uint16_t partner[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int d = 8 * u + e;
        partner[e] = d < n ? src[d < h ? d + h : d - h] : (uint16_t)0;
    }
    const uint32_t w[4] = {own.x, own.y, own.z, own.w};
    uint32_t r[4];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int d = 8 * u + e;
        const uint32_t x = e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
        uint32_t y = x;
        if (d < h) y = rot_pair(x | (uint32_t)partner[e] << 16, cs[d]) & 0xffffu;
        else if (d < n) y = rot_pair((uint32_t)partner[e] | x << 16, cs[d - h]) >> 16;
        if (e & 1) r[e >> 1] |= y << 16;
        else r[e >> 1] = y;
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// Element i of a head that is turned in place in the odd form, where nobody else may have written what a pair reads:
// i < n / 2 a pair, then the rest.
template <class Put>
__device__ __forceinline__ void rot_item(const RopeArgs &a, const uint16_t *src, int i, const float2 *cs, Put put) {
    const int h = a.rotary / 2;
    if (i >= h) {
        put(i + h, src[i + h]);
        return;
    }
    const uint32_t r = rot_pair((uint32_t)src[i] | (uint32_t)src[i + h] << 16, cs[i]);
    put(i, (uint16_t)r);
    put(i + h, (uint16_t)(r >> 16));
}

// Rotated, bf16-rounded column d of a head (Q8_0 pools quantise whole 32-column groups).
__device__ __forceinline__ float rot_at(const RopeArgs &a, const uint16_t *src, int d, const float2 *cs) {
    if (d >= a.rotary) return bf16_bits_to_f32(src[d]);
    const int h = a.rotary / 2;
    const int i = a.interleaved ? d >> 1 : d < h ? d : d - h;
    const bool second = a.interleaved ? d & 1 : d >= h;
    const uint32_t w = a.interleaved ? (uint32_t)src[2 * i] | (uint32_t)src[2 * i + 1] << 16
                                     : (uint32_t)src[i] | (uint32_t)src[i + h] << 16;
    const uint32_t r = rot_pair(w, cs[i]);
    return bf16_bits_to_f32(second ? (uint16_t)(r >> 16) : (uint16_t)r);
}

// Grid: (row chunk, request). WIDE: every head is whole 16-byte units.
template <bool Q8, bool WIDE>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const RopeArgs a) {
    extern __shared__ __align__(16) float2 s_cs[];  // [rows][rotary / 2]
    __shared__ int s_blk[kMaxRows], s_rib[kMaxRows];
    const PoolView &p = a.pool;
    decode::grid_wait();
    const int b = blockIdx.y, r0 = blockIdx.x * a.rows_per_cta;
    const int nr = min(a.rows_per_cta, min(a.max_rows, a.n_rows[b]) - r0);
    if (nr <= 0) return;
    const int half = a.rotary / 2, D = p.head_dim, wlog = decode::log2_of(p.swz_bytes);
    const int64_t row0 = (int64_t)a.src_row[b] + r0;
    if (a.k && (int)threadIdx.x < nr) {
        const int seq = a.seq_ids[b], pos = a.dst_pos[b] + r0 + (int)threadIdx.x;
        int blk = -1;
        if (seq < 0 || seq >= p.max_seqs) {
            report_error(p.status, DEV_ERR_BAD_SEQ, seq, pos, 9);
        } else if (pos < 0 || pos >= p.seq_lens[seq]) {
            report_error(p.status, DEV_ERR_BAD_POS, seq, pos, p.seq_lens[seq]);
        } else {
            blk = lookup_block(p, seq, pos / p.block_tokens);
        }
        s_blk[threadIdx.x] = blk;
        s_rib[threadIdx.x] = pos < 0 ? 0 : pos % p.block_tokens;
    }
    for (int i = threadIdx.x; i < nr * half; i += kThreads) {
        const int r = i / half, j = i - r * half;
        const double t = __dmul_rn((double)a.positions[row0 + r], a.turns[j]);
        float sn, cn;
        sincospif(2.0f * (float)(t - rint(t)), &sn, &cn);
        s_cs[i] = make_float2(cn * a.magnitude, sn * a.magnitude);
    }
    __syncthreads();
    // Items of the CTA's rows: (row, head, unit) of q, then of k, then of v, kLoads of them in flight per thread.
    const int hk = p.kv_heads;
    if (a.q) {
        const bool items = !WIDE && a.per_item > 0;
        const int per = items ? a.per_item : a.per, total = nr * a.q_heads * per;
        for (int i0 = threadIdx.x; i0 < total; i0 += kThreads * kLoads) {
            Unit x[kLoads];
            int rr[kLoads], uu[kLoads];
            int64_t at[kLoads];
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int i = i0 + j * kThreads;
                rr[j] = -1;
                if (i >= total) continue;
                const int hr = items ? a.div_item(i) : a.div_per(i), r = a.div_q(hr), h = hr - r * a.q_heads;
                rr[j] = r;
                uu[j] = i - hr * per;
                const uint16_t *src = a.q + (row0 + r) * a.q_stride + h * D;
                at[j] = ((row0 + r) * a.q_heads + h) * D;
                if (WIDE) x[j] = load_unit(a, src, uu[j]);
                else if (items) rot_item(a, src, uu[j], s_cs + r * half, [&](int d, uint16_t v) { a.q_out[at[j] + d] = v; });
                else x[j].x = odd_unit(a, src, uu[j], s_cs + r * half);
            }
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                if (rr[j] < 0 || items) continue;
                auto put = [&](int d, uint4 v) { *(uint4 *)(a.q_out + at[j] + d) = v; };
                if constexpr (WIDE) turn_unit(a, x[j], uu[j], s_cs + rr[j] * half, put);
                else put(8 * uu[j], x[j].x);
            }
        }
    }
    if (!a.k) return;
    if (Q8) {
        // the group's values as ekv_append would get them (bf16), quantised by its rule
        const int groups = D / 32, total = nr * hk * groups;
        for (int i = threadIdx.x; i < 2 * total; i += kThreads) {
            const bool is_v = i >= total;
            const int hr = (is_v ? i - total : i) / groups, u = (is_v ? i - total : i) - hr * groups;
            const int r = a.div_kv(hr), h = hr - r * hk;
            if (s_blk[r] < 0) continue;
            const uint16_t *src = (is_v ? a.v : a.k) + (row0 + r) * a.kv_stride + h * D;
            uint8_t *tile = p.prefix + prefix_tile_index(p, a.layer, s_blk[r], is_v ? 1 : 0, h) * p.tile_bytes;
            float x[32], amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                x[j] = is_v ? bf16_bits_to_f32(src[32 * u + j]) : rot_at(a, src, 32 * u + j, s_cs + r * half);
                amax = fmaxf(amax, fabsf(x[j]));
            }
            const float d = __fdiv_rn(amax, 127.0f), id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                w[j] = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[j] |= ((uint32_t)(uint8_t)(int8_t)(int)roundf(__fmul_rn(x[4 * j + e], id))) << (8 * e);
            }
            const int rib = s_rib[r];
            *(uint4 *)(tile + q8_qs_off(rib, 32 * u, D)) = make_uint4(w[0], w[1], w[2], w[3]);
            *(uint4 *)(tile + q8_qs_off(rib, 32 * u + 16, D)) = make_uint4(w[4], w[5], w[6], w[7]);
            *((uint16_t *)(tile + (int64_t)p.block_tokens * D) + rib * groups + u) = __half_as_ushort(__float2half_rn(d));
        }
        return;
    }
    const int per = a.per, total_k = nr * hk * per;
    for (int i0 = threadIdx.x; i0 < total_k; i0 += kThreads * kLoads) {
        Unit x[kLoads];
        int rr[kLoads], uu[kLoads];
        uint8_t *tile[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int i = i0 + j * kThreads;
            rr[j] = -1;
            if (i >= total_k) continue;
            const int hr = a.div_per(i), r = a.div_kv(hr), h = hr - r * hk;
            if (s_blk[r] < 0) continue;
            rr[j] = r;
            uu[j] = i - hr * per;
            const uint16_t *src = a.k + (row0 + r) * a.kv_stride + h * D;
            tile[j] = p.prefix + prefix_tile_index(p, a.layer, s_blk[r], 0, h) * p.tile_bytes;
            if (WIDE) x[j] = load_unit(a, src, uu[j]);
            else x[j].x = odd_unit(a, src, uu[j], s_cs + r * half);
        }
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            if (rr[j] < 0) continue;
            auto put = [&](int d, uint4 v) { *(uint4 *)(tile[j] + decode::bf16_off_any(s_rib[rr[j]], d, D, wlog)) = v; };
            if constexpr (WIDE) turn_unit(a, x[j], uu[j], s_cs + rr[j] * half, put);
            else put(8 * uu[j], x[j].x);
        }
    }
    const int pv = D / 8, total_v = nr * hk * pv;
    for (int i0 = threadIdx.x; i0 < total_v; i0 += kThreads * 2 * kLoads) {
        uint4 x[2 * kLoads];
        uint8_t *to[2 * kLoads];
#pragma unroll
        for (int j = 0; j < 2 * kLoads; ++j) {
            const int i = i0 + j * kThreads;
            to[j] = nullptr;
            if (i >= total_v) continue;
            const int hr = a.div_v(i), u = i - hr * pv, r = a.div_kv(hr), h = hr - r * hk;
            if (s_blk[r] < 0) continue;
            x[j] = *(const uint4 *)(a.v + (row0 + r) * a.kv_stride + h * D + 8 * u);
            to[j] = p.prefix + prefix_tile_index(p, a.layer, s_blk[r], 1, h) * p.tile_bytes + decode::bf16_off_any(s_rib[r], 8 * u, D, wlog);
        }
#pragma unroll
        for (int j = 0; j < 2 * kLoads; ++j)
            if (to[j]) *(uint4 *)to[j] = x[j];
    }
}

}  // namespace

int launch_rope_append(const PoolView &p, const ekv_rope *rope, int layer, int n_batch, const int32_t *seq_ids,
                       const int32_t *dst_pos, const int32_t *n_rows, const int32_t *src_row, int max_rows,
                       const int32_t *positions, int q_heads, const void *q, int64_t q_stride, void *q_out, const void *k,
                       const void *v, int64_t kv_stride, int sms, cudaStream_t s) {
    RopeArgs a{};
    a.pool = p;
    a.layer = layer;
    a.n_batch = n_batch;
    a.max_rows = max_rows;
    a.q_heads = q_heads;
    a.interleaved = rope->interleaved;
    a.rotary = rope->rotary;
    a.magnitude = rope->magnitude;
    a.turns = rope->dev_turns;
    a.seq_ids = seq_ids;
    a.dst_pos = dst_pos;
    a.n_rows = n_rows;
    a.src_row = src_row;
    a.positions = positions;
    a.q = (const uint16_t *)q;
    a.k = (const uint16_t *)k;
    a.v = (const uint16_t *)v;
    a.q_stride = q_stride;
    a.kv_stride = kv_stride;
    a.q_out = (uint16_t *)q_out;
    // as few rows as leave one wave of CTAs (4 per SM): a CTA's chain of dependent loads is not paid twice
    a.rows_per_cta = (int)std::min<int64_t>(kMaxRows, std::max<int64_t>(1, ((int64_t)max_rows * n_batch + 4 * sms - 1) / (4 * sms)));
    const dim3 grid((unsigned)((max_rows + a.rows_per_cta - 1) / a.rows_per_cta), (unsigned)n_batch);
    const size_t smem = (size_t)a.rows_per_cta * (a.rotary / 2) * sizeof(float2);
    const bool wide = a.interleaved || a.rotary % 16 == 0;
    const int D = p.head_dim;
    a.per = !wide || a.interleaved ? D / 8 : a.rotary / 16 + (D - a.rotary) / 8;
    a.per_item = !wide && q == q_out ? D - a.rotary / 2 : 0;
    // (as two comparisons: the whole product passes 64 bits from 2^28 heads on)
    const int64_t items = (int64_t)kMaxRows * std::max(q_heads, p.kv_heads) * D;
    if (items >= 1ll << 32 || items * std::max({a.per, a.per_item, q_heads, p.kv_heads, D / 8}) >= 1ll << 32)
        return EKV_ERR_UNSUPPORTED;
    a.div_per = SmallDiv((uint32_t)a.per);
    a.div_item = SmallDiv((uint32_t)std::max(1, a.per_item));
    a.div_q = SmallDiv((uint32_t)std::max(1, q_heads));
    a.div_kv = SmallDiv((uint32_t)p.kv_heads);
    a.div_v = SmallDiv((uint32_t)(D / 8));
    if (p.dtype == EKV_DTYPE_Q8_0) {
        if (wide) return decode::launch_after(rope_append_kernel<true, true>, grid, kThreads, smem, s, a);
        else return decode::launch_after(rope_append_kernel<true, false>, grid, kThreads, smem, s, a);
    } else {
        if (wide) return decode::launch_after(rope_append_kernel<false, true>, grid, kThreads, smem, s, a);
        else return decode::launch_after(rope_append_kernel<false, false>, grid, kThreads, smem, s, a);
    }
}

int rope_device(const ekv_rope *r) { return r->device; }
int rope_dims(const ekv_rope *r) { return r->rotary; }

}  // namespace ekv

extern "C" int ekv_rope_create(const ekv_rope_config *c, ekv_rope **out) {
    if (!c || !out) return EKV_ERR_INVALID_ARG;
    *out = nullptr;
    if (c->rotary_dims < 2 || c->rotary_dims % 2) return EKV_ERR_INVALID_ARG;
    if (c->rotary_dims > 256) return EKV_ERR_UNSUPPORTED;
    if (c->layout != EKV_ROPE_HALF && c->layout != EKV_ROPE_INTERLEAVED) return EKV_ERR_INVALID_ARG;
    if (!(c->freq_base > 1.0f) || !std::isfinite(c->freq_base) || !(c->freq_scale > 0.0f) || !std::isfinite(c->freq_scale) ||
        !std::isfinite(c->attn_factor) || !(c->ext_factor >= 0.0f && c->ext_factor <= 1.0f))
        return EKV_ERR_INVALID_ARG;
    const double n = c->rotary_dims, base = c->freq_base;
    double low = 0, high = 0;
    if (c->ext_factor != 0.0f) {
        if (c->n_ctx_orig <= 0 || !(c->beta_fast > 0.0f) || !(c->beta_slow > 0.0f)) return EKV_ERR_INVALID_ARG;
        // the pair that turns `beta` times over the trained length
        const double two_pi = 6.283185307179586476925;
        low = std::floor(n * std::log(c->n_ctx_orig / (c->beta_fast * two_pi)) / (2 * std::log(base)));
        high = std::ceil(n * std::log(c->n_ctx_orig / (c->beta_slow * two_pi)) / (2 * std::log(base)));
        low = std::max(0.0, low);
        high = std::min(n - 1, high);
    }
    ekv_rope *r = new (std::nothrow) ekv_rope();
    if (!r) return EKV_ERR_ALLOC;
    r->device = c->device;
    r->interleaved = c->layout == EKV_ROPE_INTERLEAVED;
    r->rotary = c->rotary_dims;
    r->magnitude = c->attn_factor;
    if (c->ext_factor != 0.0f) r->magnitude *= (float)(1.0 + 0.1 * std::log(1.0 / (double)c->freq_scale));
    r->dev_turns = nullptr;
    double turns[128];
    for (int i = 0; i < c->rotary_dims / 2; ++i) {
        const double ff = c->freq_factors ? (double)c->freq_factors[i] : 1.0;
        if (!(ff > 0.0) || !std::isfinite(ff)) {
            delete r;
            return EKV_ERR_INVALID_ARG;
        }
        const double f = std::pow(base, -2.0 * i / n) / ff;
        double kept = 0.0;  // the share of the unscaled frequency
        if (c->ext_factor != 0.0f)
            kept = (1.0 - std::min(1.0, std::max(0.0, (i - low) / std::max(0.001, high - low)))) * c->ext_factor;
        r->freq[i] = f * (kept + (1.0 - kept) * c->freq_scale);
        turns[i] = r->freq[i] / 6.283185307179586476925;
    }
    if (c->device >= 0) {
        int prev = 0;
        if (cudaGetDevice(&prev) != cudaSuccess || (prev != c->device && cudaSetDevice(c->device) != cudaSuccess)) {
            cudaGetLastError();
            delete r;
            return EKV_ERR_CUDA;
        }
        const size_t bytes = (size_t)(c->rotary_dims / 2) * sizeof(double);
        int rc = cudaMalloc((void **)&r->dev_turns, bytes) == cudaSuccess ? EKV_OK : EKV_ERR_ALLOC;
        // (the copy of pageable memory may return before it has landed, and other streams do not wait for this one)
        if (!rc && (cudaMemcpy(r->dev_turns, turns, bytes, cudaMemcpyHostToDevice) != cudaSuccess ||
                    cudaStreamSynchronize(cudaStreamLegacy) != cudaSuccess))
            rc = EKV_ERR_CUDA;
        if (rc && r->dev_turns) cudaFree(r->dev_turns);
        if (rc) cudaGetLastError();
        if (prev != c->device) cudaSetDevice(prev);
        if (rc) {
            delete r;
            return rc;
        }
    }
    *out = r;
    return EKV_OK;
}

extern "C" int ekv_rope_destroy(ekv_rope *r) {
    if (!r) return EKV_ERR_INVALID_ARG;
    if (r->dev_turns) {
        int prev = 0;
        const bool have = cudaGetDevice(&prev) == cudaSuccess;
        if (have && prev != r->device) cudaSetDevice(r->device);
        cudaFree(r->dev_turns);
        if (have && prev != r->device) cudaSetDevice(prev);
    }
    delete r;
    return EKV_OK;
}

extern "C" int ekv_rope_get(const ekv_rope *r, double *freq, int32_t cap, float *magnitude) {
    if (!r || cap < 0 || (cap > 0 && !freq)) return EKV_ERR_INVALID_ARG;
    for (int i = 0; i < std::min(cap, r->rotary / 2); ++i) freq[i] = r->freq[i];
    if (magnitude) *magnitude = r->magnitude;
    return EKV_OK;
}
