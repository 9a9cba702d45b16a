// ekv_norm_rope.cu -- RMS norms of the q and k heads, their rotation, and the append to the pool's pages, in one pass.
//
// For a head x of D columns: y = x / sqrt(mean(x^2) + eps) * (w + offset), and pair i of the first `rotary` columns turns by
// pos * f_i (ekv_rope.cu says how the angle is taken); the norm comes before the rotation, or after it.
// A warp has a row, or a share of its heads where the call has few rows. A head is P = D / 16 lanes' (rounded up to a power of
// two), 16 columns each, so that its sum of squares takes log2(P) shuffles and a pair's two columns are one lane's: with the split
// layout a lane has columns 8 l .. 8 l + 7 and their partners. The sines of a row are computed once per warp, a lane's pairs and
// weights stay in registers over its heads.
// Bound: instructions beside DRAM. 29 k rows of 48 heads of 128 columns (683 MB read and written) take 127 us, 5.4 TB/s, 82% of the
// measured copy rate (8-bit pages, 630 MB: 134 us, 72%), with half of the issue slots taken: 28 us of it go to what a warp does once a
// row (sines, weights, places; that much more for every further warp that a row is given). Three CTAs per SM leave 80 registers, of
// which split pairs over bf16 pages spill up to 16; four spill more (145 us), two hide less (142). Sines in registers 135, several rows a
// warp in turn 139 to 150. One row takes 5 us.
#include <algorithm>

#include "ekv_decode.cuh"

namespace ekv {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct NormRopeArgs {
    PoolView pool;
    int32_t layer, max_rows, warps_per_row, q_heads;  // warps_per_row: a power of two
    int32_t interleaved, rotary, after, weight_f32;
    float magnitude, eps, weight_offset, inv_dim;
    const double *turns;
    const void *q_weight, *k_weight;
    const int32_t *seq_ids, *dst_pos, *n_rows, *src_row, *positions;
    const uint16_t *q, *k, *v;
    int64_t q_stride, kv_stride;  // elements per source row
    uint16_t *q_out;
};

// How a lane's 16 columns lie: two runs of eight, at `a` and `b`. Split: pairs (a + i, b + i); otherwise pairs are neighbours
// (interleaved), or are found through shared memory (split pairs that are no whole runs of eight).
enum class Pairs { Split, Neighbours, Odd };

template <Pairs K>
struct Columns {
    int a, b;
    bool turns;  // Split: the lane's columns are pairs (others pass)
    __device__ __forceinline__ Columns(int l, int n) {
        a = 16 * l;
        b = a + 8;
        turns = true;
        if (K == Pairs::Split) {
            const int t = n / 16;  // lanes whose columns turn
            turns = l < t;
            if (turns) {
                a = 8 * l;
                b = n / 2 + a;
            }
        }
    }
};

// Pairs of f32 in one register: eight of them are a lane's columns.
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void unpack8(uint4 v, uint64_t *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = decode::pair_of(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ uint4 pack8(const uint64_t *x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = decode::pack_bf16(decode::of_pair(x[i]).x, decode::of_pair(x[i]).y);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 adjacent columns of a row to an 8-bit page: the rule of ekv_append (two lanes hold a group of 32).
__device__ __forceinline__ void quantise16(const uint64_t (&pairs)[8], uint8_t *tile, int rib, int col, int D, int block_tokens, bool on) {
    float x[16], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[2 * i] = decode::of_pair(pairs[i]).x;
        x[2 * i + 1] = decode::of_pair(pairs[i]).y;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    if (!on) return;
    const float d = __fdiv_rn(amax, 127.0f), id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        w[j] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[j] |= ((uint32_t)(uint8_t)(int8_t)(int)roundf(__fmul_rn(x[4 * j + e], id))) << (8 * e);
    }
    *(uint4 *)(tile + q8_qs_off(rib, col, D)) = make_uint4(w[0], w[1], w[2], w[3]);
    if (!(col & 16)) *((uint16_t *)(tile + (int64_t)block_tokens * D) + rib * (D / 32) + col / 32) = __half_as_ushort(__float2half_rn(d));
}

// Grid: (rows, request). P: lanes of a head.
template <bool Q8, int P, Pairs K>
__global__ void __launch_bounds__(kThreads, 3) norm_rope_kernel(const NormRopeArgs a) {
    constexpr int H = 32 / P;  // heads of a warp at a time
    constexpr bool kExchange = Q8 || K == Pairs::Odd;
    __shared__ __align__(16) float s_cs[kWarps][2][128];  // cosines and sines of the row's pairs
    __shared__ __align__(16) float s_x[kExchange ? kWarps : 1][kExchange ? 32 * 16 : 4];
    const PoolView &p = a.pool;
    decode::grid_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % P, sub = lane / P;
    const int share = a.warps_per_row, part = warp & (share - 1);
    const int b = blockIdx.y, r = blockIdx.x * (kWarps / share) + warp / share;
    if (r >= min(a.max_rows, a.n_rows[b])) return;
    const int64_t row = (int64_t)a.src_row[b] + r;
    const int D = p.head_dim, n = a.rotary, hk = p.kv_heads;
    const bool mine = 16 * l < D;
    const Columns<K> col(l, n);
    float *const cosine = s_cs[warp][0], *const sine = s_cs[warp][1];
    float *sx = s_x[kExchange ? warp : 0] + (kExchange ? sub * 16 * P : 0);

    // where k and v go
    int blk = -1, rib = 0;
    if (a.k) {
        const int seq = a.seq_ids[b], pos = a.dst_pos[b] + r;
        const int at = max(pos, 0), entry = p.bt_shift >= 0 ? at >> p.bt_shift : at / p.block_tokens;
        rib = at - entry * p.block_tokens;
        if (lane == 0) {
            if (seq < 0 || seq >= p.max_seqs) {
                report_error(p.status, DEV_ERR_BAD_SEQ, seq, pos, 13);
            } else if (pos < 0 || pos >= p.seq_lens[seq]) {
                report_error(p.status, DEV_ERR_BAD_POS, seq, pos, p.seq_lens[seq]);
            } else {
                blk = lookup_block_to_write(p, seq, entry);
            }
        }
        blk = __shfl_sync(0xffffffffu, blk, 0);
    }

    uint64_t w[8];
    auto load_weights = [&](const void *from) {
        const uint64_t offset = decode::pair_of(a.weight_offset, a.weight_offset);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = decode::pair_of(1.0f, 1.0f);
        if (from && mine) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int c = half ? col.b : col.a;
                if (a.weight_f32) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float4 v = __ldg((const float4 *)((const float *)from + c) + i);
                        w[4 * half + 2 * i] = decode::pair_of(v.x, v.y);
                        w[4 * half + 2 * i + 1] = decode::pair_of(v.z, v.w);
                    }
                } else {
                    unpack8(__ldg((const uint4 *)((const uint16_t *)from + c)), w + 4 * half);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = decode::add_pair(w[i], offset);
    };
    // A warp's share of the head groups; two groups' loads are on their way, the first while the sines are computed. Lanes past
    // the last head, or past its columns, read what others do.
    const int col_a = mine ? col.a : 0, col_b = mine ? col.b : 0;
    auto load = [&](const uint16_t *heads, int h, int count, uint4 (&v)[2]) {
        const uint16_t *src = heads + min(h, count - 1) * D;
        v[0] = *(const uint4 *)(src + col_a);
        v[1] = *(const uint4 *)(src + col_b);
    };
    const int h0 = part * H + sub, step = share * H;
    uint4 raw[2][2];
    {
        const uint16_t *heads = a.q ? a.q + row * a.q_stride : a.k + row * a.kv_stride;
        const int count = a.q ? a.q_heads : hk;
        load(heads, h0, count, raw[0]);
        load(heads, h0 + step, count, raw[1]);
    }

    const int at = a.positions[row];
    // (pairs that do not turn have the angle 0)
    for (int i = lane; i < 8 * P; i += 32) {
        float sn = 0.0f, cn = 1.0f;
        if (i < n / 2) {
            const double t = __dmul_rn((double)at, a.turns[i]);
            sincospif(2.0f * (float)(t - rint(t)), &sn, &cn);
            sn *= a.magnitude;
            cn *= a.magnitude;
        }
        cosine[i] = cn;
        sine[i] = sn;
    }
    __syncwarp();

    const uint64_t minus = decode::pair_of(-1.0f, -1.0f);
    auto rotate = [&](uint64_t (&x)[8]) {
        if constexpr (K == Pairs::Odd) {
            // (16 l .. 16 l + 15; partners through shared memory)
#pragma unroll
            for (int i = 0; i < 8; ++i) *(float2 *)&sx[16 * l + 2 * i] = decode::of_pair(x[i]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float y[2] = {decode::of_pair(x[i]).x, decode::of_pair(x[i]).y};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = 16 * l + 2 * i + e, h = n / 2;
                    if (d < h) y[e] = fmaf(y[e], cosine[d], -sx[d + h] * sine[d]);
                    else if (d < n) y[e] = fmaf(sx[d - h], sine[d - h], y[e] * cosine[d - h]);
                }
                x[i] = decode::pair_of(y[0], y[1]);
            }
            __syncwarp();
        } else {
            // a lane's eight pairs: columns (a + i, b + i), or (16 l + 2 i, 16 l + 2 i + 1)
            float c[8], t[8];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                *(float4 *)&c[4 * i] = *(const float4 *)&cosine[8 * l + 4 * i];
                *(float4 *)&t[4 * i] = *(const float4 *)&sine[8 * l + 4 * i];
            }
            if constexpr (K == Pairs::Split) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint64_t u = x[i], v = x[4 + i], cn = decode::pair_of(c[2 * i], c[2 * i + 1]), sn = decode::pair_of(t[2 * i], t[2 * i + 1]);
                    x[i] = decode::fma_pair(mul_pair(v, sn), minus, mul_pair(u, cn));
                    x[4 + i] = decode::fma_pair(u, sn, mul_pair(v, cn));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 v = decode::of_pair(x[i]);
                    x[i] = decode::pair_of(fmaf(v.x, c[i], -v.y * t[i]), fmaf(v.x, t[i], v.y * c[i]));
                }
            }
        }
    };
    // A head's factor 1 / sqrt(mean + eps) is taken with the last product: it and the rotation do not mind their order.
    auto factor = [&](const uint64_t (&x)[8]) {
        uint64_t s0 = 0, s1 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s0 = decode::fma_pair(x[i], x[i], s0);
            s1 = decode::fma_pair(x[4 + i], x[4 + i], s1);
        }
        const float2 t = decode::of_pair(decode::add_pair(s0, s1));
        float s = mine ? t.x + t.y : 0.0f;
#pragma unroll
        for (int o = 1; o < P; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const float f = rsqrtf(fmaf(s, a.inv_dim, a.eps));
        return decode::pair_of(f, f);
    };
    auto whole = [&](const uint4 (&v)[2], uint64_t (&x)[8]) {
        unpack8(v[0], x);
        unpack8(v[1], x + 4);
        if (a.after) rotate(x);
        const uint64_t f = factor(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = mul_pair(x[i], w[i]);
        if (!a.after) rotate(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = mul_pair(x[i], f);
    };

    if (a.q) {
        const uint16_t *q = a.q + row * a.q_stride;
        uint16_t *const to = a.q_out + row * a.q_heads * D;
        load_weights(a.q_weight);
        auto turn_q = [&](const uint4 (&v)[2], int h) {
            uint64_t x[8];
            whole(v, x);
            if (mine && h < a.q_heads) {
                *(uint4 *)(to + h * D + col.a) = pack8(x);
                *(uint4 *)(to + h * D + col.b) = pack8(x + 4);
            }
        };
#pragma unroll 1
        for (int h = h0; h - sub < a.q_heads; h += 2 * step) {
            turn_q(raw[0], h);
            load(q, h + 2 * step, a.q_heads, raw[0]);
            if (h + step - sub >= a.q_heads) break;
            turn_q(raw[1], h + step);
            load(q, h + 3 * step, a.q_heads, raw[1]);
        }
        if (a.k) {
            const uint16_t *k = a.k + row * a.kv_stride;
            load(k, h0, hk, raw[0]);
            load(k, h0 + step, hk, raw[1]);
        }
    }
    if (blk < 0) return;  // no k, or a row that was reported
    const int wlog = decode::log2_of(p.swz_bytes);
    uint8_t *const tiles = p.prefix + prefix_tile_index(p, a.layer, blk, 0, 0) * p.tile_bytes;
    const uint16_t *k = a.k + row * a.kv_stride, *v = a.v + row * a.kv_stride + (mine ? 16 * l : 0);
    uint4 vraw[2];
    auto load_v = [&](int h) {
        const uint4 *src = (const uint4 *)(v + min(h, hk - 1) * D);
        vraw[0] = src[0];
        vraw[1] = src[1];
    };
    load_v(h0);
    load_weights(a.k_weight);
    const uint32_t off_a = decode::bf16_off_any(rib, col.a, D, wlog), off_b = decode::bf16_off_any(rib, col.b, D, wlog);
    auto turn_k = [&](const uint4 (&r)[2], int h) {
        uint64_t x[8];
        whole(r, x);
        const bool on = mine && h < hk;
        uint8_t *tile = tiles + (on ? h : 0) * p.tile_bytes;
        if constexpr (!Q8) {
            if (on) {
                *(uint4 *)(tile + off_a) = pack8(x);
                *(uint4 *)(tile + off_b) = pack8(x + 4);
            }
        } else {
            // rounded to bf16 as ekv_append would get them, and in their natural order, 16 adjacent columns a lane
            uint4 *buf = (uint4 *)sx;
            if (mine) {
                buf[col.a / 8] = pack8(x);
                buf[col.b / 8] = pack8(x + 4);
            }
            __syncwarp();
            if (mine) {
                unpack8(buf[2 * l], x);
                unpack8(buf[2 * l + 1], x + 4);
            }
            quantise16(x, tile, rib, 16 * l, D, p.block_tokens, on);
            __syncwarp();
        }
    };
#pragma unroll 1
    for (int h = h0; h - sub < hk; h += 2 * step) {
        turn_k(raw[0], h);
        load(k, h + 2 * step, hk, raw[0]);
        if (h + step - sub >= hk) break;
        turn_k(raw[1], h + step);
        load(k, h + 3 * step, hk, raw[1]);
    }
    const uint32_t off_v = decode::bf16_off_any(rib, 16 * l, D, wlog);  // (the next eight columns are the neighbouring unit)
#pragma unroll 1
    for (int h = h0; h - sub < hk; h += step) {
        const bool on = mine && h < hk;
        uint8_t *tile = tiles + (hk + (on ? h : 0)) * p.tile_bytes;
        if constexpr (!Q8) {
            if (on) {
                *(uint4 *)(tile + off_v) = vraw[0];
                *(uint4 *)(tile + (off_v ^ 16u)) = vraw[1];
            }
        } else {
            uint64_t x[8];
            unpack8(vraw[0], x);
            unpack8(vraw[1], x + 4);
            quantise16(x, tile, rib, 16 * l, D, p.block_tokens, on);
        }
        load_v(h + step);
    }
}

template <bool Q8, int P>
int launch_pairs(const NormRopeArgs &a, dim3 grid, cudaStream_t s) {
    if (a.interleaved) return decode::launch_after(norm_rope_kernel<Q8, P, Pairs::Neighbours>, grid, kThreads, 0, s, a);
    if (a.rotary % 16 == 0) return decode::launch_after(norm_rope_kernel<Q8, P, Pairs::Split>, grid, kThreads, 0, s, a);
    return decode::launch_after(norm_rope_kernel<Q8, P, Pairs::Odd>, grid, kThreads, 0, s, a);
}
template <bool Q8>
int launch_lanes(const NormRopeArgs &a, dim3 grid, cudaStream_t s) {
    const int lanes = a.pool.head_dim / 16;
    if (lanes <= 1) return Q8 ? EKV_ERR_UNSUPPORTED : launch_pairs<false, 1>(a, grid, s);
    if (lanes <= 2) return launch_pairs<Q8, 2>(a, grid, s);
    if (lanes <= 4) return launch_pairs<Q8, 4>(a, grid, s);
    if (lanes <= 8) return launch_pairs<Q8, 8>(a, grid, s);
    return launch_pairs<Q8, 16>(a, grid, s);
}

}  // namespace

int launch_norm_rope_append(const PoolView &p, const ekv_rope *rope, const ekv_head_norm *norm, int layer, int n_batch,
                            const int32_t *seq_ids, const int32_t *dst_pos, const int32_t *n_rows, const int32_t *src_row, int max_rows,
                            const int32_t *positions, int q_heads, const void *q, int64_t q_stride, void *q_out, const void *k,
                            const void *v, int64_t kv_stride, int sms, cudaStream_t s) {
    NormRopeArgs a{};
    a.pool = p;
    a.layer = layer;
    a.max_rows = max_rows;
    a.q_heads = q ? q_heads : 0;
    a.interleaved = rope->interleaved;
    a.rotary = rope->rotary;
    a.after = norm->after_rotation != 0;
    a.weight_f32 = norm->weight_dtype == EKV_DTYPE_F32;
    a.magnitude = rope->magnitude;
    a.eps = norm->eps;
    a.weight_offset = norm->weight_offset;
    a.inv_dim = 1.0f / (float)p.head_dim;
    a.turns = rope->dev_turns;
    a.q_weight = norm->q_weight;
    a.k_weight = norm->k_weight;
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
    if (std::max<int64_t>(q_heads, p.kv_heads) * p.head_dim >= 1 << 30) return EKV_ERR_UNSUPPORTED;
    // a row's heads are shared by warps until there are sixteen warps an SM
    a.warps_per_row = 1;
    while (a.warps_per_row < kWarps && (int64_t)max_rows * n_batch * a.warps_per_row < 16ll * sms) a.warps_per_row *= 2;
    const int rows = kWarps / a.warps_per_row;
    const dim3 grid((unsigned)((max_rows + rows - 1) / rows), (unsigned)n_batch);
    return p.dtype == EKV_DTYPE_Q8_0 ? launch_lanes<true>(a, grid, s) : launch_lanes<false>(a, grid, s);
}

}  // namespace ekv
