// ekv_tree.cu -- attention of a tree of drafted tokens over the paged cache (one token: plain decoding).
//
// For request b, drafted token t and query head h (KV head h / group), over the cached keys and those
// drafted keys that t's ancestor word names:
//   s_k = scale * q.k  (or cap * tanh(scale * q.k / cap)),  out = sum exp(s_k - m) v_k / sum exp(s_k - m),
//   lse = m + ln sum exp(s_k - m).
// One pass over the keys: a warp keeps the running maximum m, the sum and the output of its 16 rows in
// registers (flash attention's recurrence, Dao et al. 2022; Milakov and Gimelshein 2018 for the softmax).
#include <algorithm>

#include "ekv_decode.cuh"

namespace ekv {
namespace {

using namespace decode;
using namespace sm100;

constexpr int kXCols = 32;  // columns that the key groups' outputs are joined in at a time

// CTAs per SM: two where a thread's share of the output (16 * MT rows by D columns over a warp) leaves the
// registers for it.
constexpr int rows_ctas(int d, int mt) { return d / 2 * mt > 64 ? 1 : 2; }

// WR row groups of 16 * MT rows times WK groups of 64 / WK keys: one warp each, and one feeder warp.
template <int D, bool Q8, int MT, int WR, int WK>
struct Cfg {
    using T = TileCfg<D, Q8>;
    static constexpr int NW = WR * WK, NC = NW * 32, THREADS = NC + 32;
    static constexpr int ROWS = 16 * MT * WR;
    static constexpr int KPW = kTile / WK;          // keys of a tile per warp
    static constexpr int NB = KPW / 16;             // 16-key steps per warp and tile
    // drafted keys per tile: bf16 rows in the tile's own layout, or padded rows where the tile is Q8_0
    static constexpr int DT = Q8 ? 32 : kTile;
    static constexpr int DROW = 2 * D + 16;         // bytes of a drafted row in a Q8_0 kernel
    static constexpr int STAGE_MIN = 2 * T::KV_BYTES, STAGE_DRAFT = Q8 ? 2 * DT * DROW : 0;
    static constexpr int STAGE = ((STAGE_MIN > STAGE_DRAFT ? STAGE_MIN : STAGE_DRAFT) + 1023) / 1024 * 1024;
    static constexpr int V_OFF = T::KV_BYTES, DRAFT_V_OFF = Q8 ? DT * DROW : T::KV_BYTES;
    static constexpr int X_BYTES = WK * ROWS * kXCols * 4;
    static constexpr int ML_BYTES = WK * ROWS * 8;
    static constexpr int FIXED = X_BYTES + ML_BYTES + 1024 + 1024;
    // two CTAs per SM where the rows' state leaves registers for it
    static constexpr int CTAS = rows_ctas(D, MT);
    static constexpr int BUDGET = CTAS == 2 ? 112 * 1024 : 220 * 1024;
    static constexpr int NST_FIT = (BUDGET - FIXED) / STAGE;
    static constexpr int NST = NST_FIT > 8 ? 8 : NST_FIT;
    static constexpr int SMEM = NST * STAGE + FIXED;
    static_assert(NST >= 2, "two stages");
};

template <int NST>
struct Shared {
    uint64_t full_k[NST], full_v[NST], empty[NST];
    unsigned long long bad[NST];  // drafted keys of the stage whose values are not all finite
    RangeScratch range;
    int abort;
};

// Column of output accumulator (n-tile nt, element i) of lane c in its quad.
template <bool Q8>
__device__ __forceinline__ int o_col(int nt, int c, int i) {
    return Q8 ? 32 * (nt >> 2) + 8 * c + 4 * (i & 1) + (nt & 3) : 8 * nt + 2 * c + (i & 1);
}

template <int D, bool Q8, int MT, int WR, int WK>
__global__ void __launch_bounds__(Cfg<D, Q8, MT, WR, WK>::THREADS, Cfg<D, Q8, MT, WR, WK>::CTAS)
    tree_rows_kernel(const TreeArgs a) {
    using C = Cfg<D, Q8, MT, WR, WK>;
    constexpr int NST = C::NST, KS = D / 16, NT = D / 8;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float *xb = (float *)(smem + NST * C::STAGE);                   // [WK][ROWS][kXCols]
    float2 *sml = (float2 *)(smem + NST * C::STAGE + C::X_BYTES);   // [WK][ROWS]
    using Sh = Shared<NST>;
    static_assert(sizeof(Sh) <= 1024, "barrier block");
    Sh &sh = *(Sh *)(smem + NST * C::STAGE + C::X_BYTES + C::ML_BYTES);
    volatile int *abort = &sh.abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hk = a.pool.kv_heads, units_per_req = hk * a.row_tiles;
    const int rows_all = a.n_draft * a.group;

    if (threadIdx.x == 0) {
        for (int i = 0; i < NST; ++i) {
            mbar_init(smem_addr(&sh.full_k[i]), 1);
            mbar_init(smem_addr(&sh.full_v[i]), 1);
            mbar_init(smem_addr(&sh.empty[i]), C::NW);
            sh.bad[i] = 0;
        }
        sh.abort = 0;
        mbar_init_fence();
    }
    // a unit without keys keeps one (empty) tile, so that some CTA writes its rows
    auto unit_tiles = [](const Req &r) {
        return max(1, (r.n_prefix + kTile - 1) / kTile + (r.n_nodes + C::DT - 1) / C::DT);
    };
    Range rg;
    if (a.split) {
        rg = find_range<C::THREADS>(a.n_batch, units_per_req, sh.range,
                                    [&](int b) { return unit_tiles(load_req(a, b, false)); });
    } else {
        __syncthreads();
        rg.b = blockIdx.x / units_per_req;
        const int n = unit_tiles(load_req(a, rg.b, false));
        rg.base = 0;
        rg.lo = (long long)(blockIdx.x - rg.b * units_per_req) * n;
        rg.hi = rg.lo + n;
        rg.total = 0;
        rg.ctas = 0;
    }

    int it = 0;  // tile counter of the CTA: stage it % NST, use it / NST
    bool ok = true;
    int b = rg.b;
    long long base = rg.base;
    for (long long x = rg.lo; x < rg.hi && b < a.n_batch;) {
        const Req rq = load_req(a, b, warp == 0);
        const int n_tiles = unit_tiles(rq);
        const long long span = (long long)n_tiles * units_per_req;
        if (x >= base + span) {
            base += span;
            ++b;
            continue;
        }
        const int u = (int)((x - base) / n_tiles);
        const int t0 = (int)((x - base) - (long long)u * n_tiles);
        const int t1 = (int)min((long long)n_tiles, t0 + (rg.hi - x));
        const int g = u / a.row_tiles, row0 = (u - g * a.row_tiles) * C::ROWS;
        const int rows = min(C::ROWS, rows_all - row0);
        const int p_tiles = (rq.n_prefix + kTile - 1) / kTile;
        const long long kv_row = ((long long)b * a.n_draft * hk + g) * D;  // drafted token 0 of this head

        if (warp == C::NW) {
            // ---- feeder ----
            Piece next = find_piece<D, Q8>(a, rq, g, t0 * kTile, lane);
            for (int j = t0; j < t1; ++j, ++it) {
                const int st = it % NST;
                const Piece pc = next;
                if (j + 1 < min(t1, p_tiles)) next = find_piece<D, Q8>(a, rq, g, (j + 1) * kTile, lane);
                if (it >= NST)
                    ok = ok && mbar_wait(smem_addr(&sh.empty[st]), ((it / NST) - 1) & 1, abort, kWait);
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                const uint32_t sk = smem_addr(smem + st * C::STAGE);
                const uint32_t bk = smem_addr(&sh.full_k[st]), bv = smem_addr(&sh.full_v[st]);
                if (j < p_tiles) {
                    issue_piece<D, Q8, true>(a, pc, sk, sk + C::V_OFF, bk, bv, lane);
                    continue;
                }
                // drafted rows, from the caller's buffers
                const int d0 = (j - p_tiles) * C::DT;
                const int n = min(C::DT, rq.n_nodes - d0);
                constexpr int U = D / 8;
                for (int i = lane; i < n * U; i += 32) {
                    const int r = i / U, col = (i - r * U) * 8;
                    const long long src = kv_row + (long long)(d0 + r) * hk * D + col;
                    const uint32_t off = Q8 ? (uint32_t)(r * C::DROW + col * 2) : bf16_off<D>(r, col);
                    cp_async_16(sk + off, a.k_draft + src);
                    cp_async_16(sk + C::DRAFT_V_OFF + off, a.v_draft + src);
                }
                cp_async_wait_all();
                // A drafted key that a row may not see must not reach it: 0 * inf would. Values that are
                // not finite leave the tile here, and rows that see their key add them one by one.
                unsigned long long bad = 0;
                for (int i = lane; i < n * U; i += 32) {
                    const int r = i / U, col = (i - r * U) * 8;
                    const uint32_t off = Q8 ? (uint32_t)(r * C::DROW + col * 2) : bf16_off<D>(r, col);
                    uint16_t *w = (uint16_t *)(smem + st * C::STAGE + C::DRAFT_V_OFF + off);
                    const uint4 v = *(const uint4 *)w;
                    const uint32_t ww[4] = {v.x, v.y, v.z, v.w};
                    bool any = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        any = any || (ww[e] & 0x7f80u) == 0x7f80u || (ww[e] & 0x7f800000u) == 0x7f800000u;
                    if (any) {
                        bad |= 1ull << r;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if ((w[e] & 0x7f80u) == 0x7f80u) w[e] = 0;
                    }
                }
                const uint32_t blo = __reduce_or_sync(0xffffffffu, (uint32_t)bad);
                const uint32_t bhi = __reduce_or_sync(0xffffffffu, (uint32_t)(bad >> 32));
                if (lane == 0) sh.bad[st] = (unsigned long long)bhi << 32 | blo;
                fence_proxy_async();  // the stage's next contents come through the copy engine
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bk);
                    mbar_arrive(bv);
                }
            }
        } else {
            // ---- rows ----
            const int wr = warp / WK, wk = warp % WK;
            const int rq0 = lane >> 2, c = lane & 3;
            // query fragments: rows row0 + (wr * MT + m) * 16 + rq0 (+ 8)
            uint32_t qf[MT][KS][4];
            int t_of[MT][2];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = row0 + (wr * MT + m) * 16 + rq0 + 8 * h;
                    const int t = r / a.group;
                    const bool on = r < rows_all && t < rq.n_nodes;
                    t_of[m][h] = on ? t : -1;
                    const uint16_t *src =
                        a.q + (((long long)b * a.n_draft + t) * a.q_heads + g * a.group + (r - t * a.group)) * D;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int half = 0; half < 2; ++half)
                            qf[m][ks][h + 2 * half] = on ? __ldg((const uint32_t *)(src + q_col<Q8>(ks, c, half))) : 0u;
                }
            float o[MT][NT][4];
            float mx[MT][2], sum[MT][2];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                mx[m][0] = mx[m][1] = -INFINITY;
                sum[m][0] = sum[m][1] = 0.0f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[m][nt][i] = 0.0f;
            }
            const ScoreFn score{a.scale_log2, a.cap_log2, a.cap_in};

            for (int j = t0; j < t1; ++j, ++it) {
                const int st = it % NST, par = (it / NST) & 1;
                uint8_t *tile = smem + st * C::STAGE;
                const uint32_t sk = smem_addr(tile);
                const bool draft = j >= p_tiles;
                const int d0 = (j - p_tiles) * C::DT;
                const int valid = draft ? min(C::DT, rq.n_nodes - d0) : min(kTile, rq.n_prefix - j * kTile);
                const bool full = !draft && valid == kTile;
                const uint32_t sv = sk + (draft ? C::DRAFT_V_OFF : C::V_OFF);
                ok = ok && mbar_wait(smem_addr(&sh.full_k[st]), par, abort, kWait);
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                bool v_ready = false;
#pragma unroll 1
                for (int kb = 0; kb < C::NB; ++kb) {
                    const int key0 = wk * C::KPW + kb * 16;  // 16 keys of the tile
                    if (key0 >= valid) break;
                    // ---- S = Q K^T ----
                    float s[MT][2][4];
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[m][n][i] = 0.0f;
                    if constexpr (!Q8) {
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) {
                            uint32_t kf[4];
                            load_k_step<D>(sk, key0, ks, lane, kf);
#pragma unroll
                            for (int m = 0; m < MT; ++m) {
                                mma_bf16(s[m][0], qf[m][ks], kf[0], kf[1]);
                                mma_bf16(s[m][1], qf[m][ks], kf[2], kf[3]);
                            }
                        }
                    } else if (draft) {
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int ks = 0; ks < KS; ++ks) {
                                const uint2 w = lds64(sk + (key0 + 8 * n + rq0) * C::DROW + 2 * q_col<true>(ks, c, 0));
#pragma unroll
                                for (int m = 0; m < MT; ++m) mma_bf16(s[m][n], qf[m][ks], w.x, w.y);
                            }
                    } else {
                        // integer products of a 32-column group are exact; its two scales join in f32
                        using T = TileCfg<D, true>;
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const int row = key0 + 8 * n + rq0, krow = key0 + 8 * n + 2 * c;
#pragma unroll
                            for (int gr = 0; gr < T::G32; ++gr) {
                                const uint2 w = lds64(sk + q8_qs_off(row, 32 * gr + 8 * c, D));
                                uint32_t k0, k1, k2, k3;
                                int8x4_to_bf16(w.x, k0, k1);
                                int8x4_to_bf16(w.y, k2, k3);
                                const float sc0 = lds_f16(sk + T::SCALES + (krow * T::G32 + gr) * 2);
                                const float sc1 = lds_f16(sk + T::SCALES + ((krow + 1) * T::G32 + gr) * 2);
#pragma unroll
                                for (int m = 0; m < MT; ++m) {
                                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                    mma_bf16(acc, qf[m][2 * gr], k0, k1);
                                    mma_bf16(acc, qf[m][2 * gr + 1], k2, k3);
                                    s[m][n][0] = fmaf(acc[0], sc0, s[m][n][0]);
                                    s[m][n][1] = fmaf(acc[1], sc1, s[m][n][1]);
                                    s[m][n][2] = fmaf(acc[2], sc0, s[m][n][2]);
                                    s[m][n][3] = fmaf(acc[3], sc1, s[m][n][3]);
                                }
                            }
                        }
                    }
                    // ---- mask, running maximum, exponentials ----
                    uint32_t vis[MT][2];  // bit k: key0 + k visible to the row
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            vis[m][h] = 0xffffu;
                            if (!full) {
                                uint64_t w = valid >= 64 ? ~0ull : (1ull << valid) - 1;
                                if (draft) {
                                    const int t = t_of[m][h];
                                    w &= t < 0 ? 0ull
                                         : a.ancestors ? __ldg(a.ancestors + (long long)b * a.n_draft + t) >> d0
                                                       : (t >= 63 ? ~0ull : (2ull << t) - 1) >> d0;
                                }
                                vis[m][h] = (uint32_t)(w >> key0) & 0xffffu;
                            }
                        }
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        float tm[2] = {-INFINITY, -INFINITY};
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float v = score(s[m][n][i]);
                                if (!full && !((vis[m][i >> 1] >> (8 * n + 2 * c + (i & 1))) & 1u)) v = -INFINITY;
                                s[m][n][i] = v;
                                tm[i >> 1] = fmaxf(tm[i >> 1], v);
                            }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            tm[h] = fmaxf(tm[h], __shfl_xor_sync(0xffffffffu, tm[h], 1));
                            tm[h] = fmaxf(tm[h], __shfl_xor_sync(0xffffffffu, tm[h], 2));
                        }
                        const float m0 = fmaxf(mx[m][0], tm[0]), m1 = fmaxf(mx[m][1], tm[1]);
                        const float u0 = m0 == -INFINITY ? 0.0f : m0, u1 = m1 == -INFINITY ? 0.0f : m1;
                        if (__any_sync(0xffffffffu, m0 != mx[m][0] || m1 != mx[m][1])) {
                            const float f0 = ex2(mx[m][0] - u0), f1 = ex2(mx[m][1] - u1);
                            sum[m][0] *= f0;
                            sum[m][1] *= f1;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                o[m][nt][0] *= f0;
                                o[m][nt][1] *= f0;
                                o[m][nt][2] *= f1;
                                o[m][nt][3] *= f1;
                            }
                            mx[m][0] = m0;
                            mx[m][1] = m1;
                        }
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            s[m][n][0] = ex2(s[m][n][0] - u0);
                            s[m][n][1] = ex2(s[m][n][1] - u0);
                            s[m][n][2] = ex2(s[m][n][2] - u1);
                            s[m][n][3] = ex2(s[m][n][3] - u1);
                            sum[m][0] += s[m][n][0] + s[m][n][1];
                            sum[m][1] += s[m][n][2] + s[m][n][3];
                        }
                    }
                    // ---- O += P V ----
                    if (!v_ready) {
                        ok = mbar_wait(smem_addr(&sh.full_v[st]), par, abort, kWait);
                        if (!ok) {
                            *abort = 1;
                            break;
                        }
                        v_ready = true;
                    }
                    if (key0 + 16 > valid) {
                        // rows past the last key hold whatever was there: 0 * that must be 0
                        const int r1 = key0 + 16;
                        if (Q8 && !draft) {
                            constexpr int G = TileCfg<D, true>::G32 > 0 ? TileCfg<D, true>::G32 : 1;
                            for (int i = valid * G + lane; i < r1 * G; i += 32)
                                *(uint16_t *)(tile + C::V_OFF + TileCfg<D, Q8>::SCALES + i * 2) = 0;
                        } else {
                            constexpr int U = D / 8;
                            for (int i = valid * U + lane; i < r1 * U; i += 32) {
                                const int r = i / U, col = (i - r * U) * 8;
                                sts128(sv + (Q8 ? (uint32_t)(r * C::DROW + col * 2) : bf16_off<D>(r, col)),
                                       make_uint4(0, 0, 0, 0));
                            }
                        }
                        fence_proxy_async();
                        __syncwarp();
                    }
                    if constexpr (!Q8) {
                        uint32_t p[MT][4];
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            p[m][0] = pack_bf16(s[m][0][0], s[m][0][1]);
                            p[m][1] = pack_bf16(s[m][0][2], s[m][0][3]);
                            p[m][2] = pack_bf16(s[m][1][0], s[m][1][1]);
                            p[m][3] = pack_bf16(s[m][1][2], s[m][1][3]);
                        }
#pragma unroll
                        for (int ds = 0; ds < KS; ++ds) {
                            uint32_t vf[4];
                            load_v_step<D>(sv, key0, ds, lane, vf);
#pragma unroll
                            for (int m = 0; m < MT; ++m) {
                                mma_bf16(o[m][2 * ds], p[m], vf[0], vf[1]);
                                mma_bf16(o[m][2 * ds + 1], p[m], vf[2], vf[3]);
                            }
                        }
                    } else {
                        const int kr[4] = {key0 + 2 * c, key0 + 2 * c + 1, key0 + 2 * c + 8, key0 + 2 * c + 9};
#pragma unroll
                        for (int gr = 0; gr < D / 32; ++gr) {
                            uint32_t b0[4], b1[4];  // operands of the group's four 8-column tiles
                            float sc[4] = {1.0f, 1.0f, 1.0f, 1.0f};
                            if (draft) {
                                uint2 w[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) w[k] = lds64(sv + kr[k] * C::DROW + (32 * gr + 4 * rq0) * 2);
                                b0[0] = __byte_perm(w[0].x, w[1].x, 0x5410);
                                b0[1] = __byte_perm(w[0].x, w[1].x, 0x7632);
                                b0[2] = __byte_perm(w[0].y, w[1].y, 0x5410);
                                b0[3] = __byte_perm(w[0].y, w[1].y, 0x7632);
                                b1[0] = __byte_perm(w[2].x, w[3].x, 0x5410);
                                b1[1] = __byte_perm(w[2].x, w[3].x, 0x7632);
                                b1[2] = __byte_perm(w[2].y, w[3].y, 0x5410);
                                b1[3] = __byte_perm(w[2].y, w[3].y, 0x7632);
                            } else {
                                uint32_t w[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    w[k] = lds32(sv + q8_qs_off(kr[k], 32 * gr + 4 * rq0, D));
                                    sc[k] = lds_f16(sv + TileCfg<D, Q8>::SCALES + (kr[k] * (D / 32) + gr) * 2);
                                }
                                int8x4_to_bf16(__byte_perm(w[0], w[1], 0x5140), b0[0], b0[1]);
                                int8x4_to_bf16(__byte_perm(w[0], w[1], 0x7362), b0[2], b0[3]);
                                int8x4_to_bf16(__byte_perm(w[2], w[3], 0x5140), b1[0], b1[1]);
                                int8x4_to_bf16(__byte_perm(w[2], w[3], 0x7362), b1[2], b1[3]);
                            }
                            // the values' scales ride on the probabilities, which are rounded once either way
#pragma unroll
                            for (int m = 0; m < MT; ++m) {
                                const uint32_t p[4] = {pack_bf16(s[m][0][0] * sc[0], s[m][0][1] * sc[1]),
                                                       pack_bf16(s[m][0][2] * sc[0], s[m][0][3] * sc[1]),
                                                       pack_bf16(s[m][1][0] * sc[2], s[m][1][1] * sc[3]),
                                                       pack_bf16(s[m][1][2] * sc[2], s[m][1][3] * sc[3])};
#pragma unroll
                                for (int e = 0; e < 4; ++e) mma_bf16(o[m][4 * gr + e], p, b0[e], b1[e]);
                            }
                        }
                    }
                    if (draft) {
                        uint32_t bad = (uint32_t)(sh.bad[st] >> key0) & 0xffffu;
                        while (bad) {  // rare: drafted values that are not finite, for the rows that see them
                            const int k = __ffs(bad) - 1;
                            bad &= bad - 1;
                            const uint16_t *v = a.v_draft + kv_row + (long long)(d0 + key0 + k) * hk * D;
#pragma unroll
                            for (int m = 0; m < MT; ++m) {
                                float pk[2];
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    float mine = 0.0f;
#pragma unroll
                                    for (int n = 0; n < 2; ++n)
#pragma unroll
                                        for (int e = 0; e < 2; ++e)
                                            if (8 * n + 2 * c + e == k) mine = s[m][n][2 * h + e];
                                    pk[h] = __shfl_sync(0xffffffffu, mine, (lane & ~3) | ((k & 7) >> 1));
                                }
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        const float x = bf16_bits_to_f32(__ldg(v + o_col<Q8>(nt, c, i)));
                                        if (!isfinite(x) && ((vis[m][i >> 1] >> k) & 1u))
                                            o[m][nt][i] = fmaf(pk[i >> 1], x, o[m][nt][i]);
                                    }
                            }
                        }
                    }
                }
                if (ok && !v_ready) {  // no key of this tile is the warp's: still stay in step with the stage
                    ok = mbar_wait(smem_addr(&sh.full_v[st]), par, abort, kWait);
                    if (!ok) *abort = 1;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&sh.empty[st]));
            }

            // ---- join the key groups, write the rows ----
            float scale_o[MT][2], l_tot[MT][2], m_tot[MT][2];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float l = sum[m][h];
                    l += __shfl_xor_sync(0xffffffffu, l, 1);
                    l += __shfl_xor_sync(0xffffffffu, l, 2);
                    if (c == 0) sml[wk * C::ROWS + (wr * MT + m) * 16 + rq0 + 8 * h] = make_float2(mx[m][h], l);
                }
            asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = (wr * MT + m) * 16 + rq0 + 8 * h;
                    float mt = -INFINITY, lt = 0.0f;
#pragma unroll
                    for (int w = 0; w < WK; ++w) mt = fmaxf(mt, sml[w * C::ROWS + r].x);
                    const float mu = mt == -INFINITY ? 0.0f : mt;
#pragma unroll
                    for (int w = 0; w < WK; ++w) {
                        const float2 ml = sml[w * C::ROWS + r];
                        lt += ml.y * ex2(ml.x - mu);
                    }
                    m_tot[m][h] = mt;
                    l_tot[m][h] = lt;
                    scale_o[m][h] = ex2(mx[m][h] - mu);
                }
            const bool whole = t0 == 0 && t1 == n_tiles;
            const long long slot = 2ll * blockIdx.x + (t0 == 0 ? 1 : 0);
            if (wk == 0 && c == 0) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = (wr * MT + m) * 16 + rq0 + 8 * h;
                        if (r >= rows) continue;
                        if (whole) {
                            if (a.lse) {
                                const int t = (row0 + r) / a.group, hq = g * a.group + (row0 + r) - t * a.group;
                                const bool none = t_of[m][h] < 0 || l_tot[m][h] == 0.0f;
                                a.lse[((long long)b * a.n_draft + t) * a.q_heads + hq] =
                                    none ? -INFINITY : (m_tot[m][h] + __log2f(l_tot[m][h])) * 0.6931471805599453f;
                            }
                        } else {
                            a.ws_ml[slot * C::ROWS + r] = make_float2(t_of[m][h] < 0 ? -INFINITY : m_tot[m][h],
                                                                      t_of[m][h] < 0 ? 0.0f : l_tot[m][h]);
                        }
                    }
            }
            if (a.split && threadIdx.x == 0 && t0 == 0) {
                const long long unit0 = base + (long long)u * n_tiles, last = unit0 + n_tiles - 1;
                a.parts[b * units_per_req + u] =
                    make_int2(blockIdx.x, (int)(((last + 1) * rg.ctas - 1) / rg.total));
            }
            // rows' final factor: 1 / sum for whole units, none for parts
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (whole) scale_o[m][h] = l_tot[m][h] == 0.0f ? 0.0f : scale_o[m][h] / l_tot[m][h];
                }
#pragma unroll
            for (int cc = 0; cc < (D + kXCols - 1) / kXCols; ++cc) {
                const int cols = min(kXCols, D - cc * kXCols);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n4 = 0; n4 < 4; ++n4) {
                        const int nt = cc * 4 + n4;
                        if (nt >= NT) continue;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = (wr * MT + m) * 16 + rq0 + 8 * (i >> 1);
                            const int col = o_col<Q8>(nt, c, i) - cc * kXCols;
                            // a row without keys of this warp has factor 0 (or 0 / 0 were there none at all)
                            const float v = mx[m][i >> 1] == -INFINITY ? 0.0f : o[m][nt][i] * scale_o[m][i >> 1];
                            xb[(wk * C::ROWS + r) * kXCols + ((col + 4 * r) & (kXCols - 1))] = v;
                        }
                    }
                asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
                for (int i = threadIdx.x; i < rows * (cols / 4); i += C::NC) {
                    const int r = i / (cols / 4), col = (i - r * (cols / 4)) * 4;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < WK; ++w) {
                        const float4 y = *(const float4 *)&xb[(w * C::ROWS + r) * kXCols + ((col + 4 * r) & (kXCols - 1))];
                        v.x += y.x;
                        v.y += y.y;
                        v.z += y.z;
                        v.w += y.w;
                    }
                    if (!whole) {
                        *(float4 *)(a.ws_o + (slot * C::ROWS + r) * D + cc * kXCols + col) = v;
                        continue;
                    }
                    const int t = (row0 + r) / a.group, hq = g * a.group + (row0 + r) - t * a.group;
                    if (t >= rq.n_nodes) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    const long long dst = (((long long)b * a.n_draft + t) * a.q_heads + hq) * D + cc * kXCols + col;
                    if (a.out_dtype == EKV_DTYPE_F32)
                        *(float4 *)((float *)a.out + dst) = v;
                    else
                        *(uint2 *)((uint16_t *)a.out + dst) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
                }
                asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
            }
        }
        x += t1 - t0;
    }
    if (!ok && lane == 0) report_error(a.pool.status, DEV_ERR_TIMEOUT, blockIdx.x, warp, 7);
    if (warp == C::NW && !ok && lane == 0) {
        // leave no copy writing this CTA's shared memory: the last uses of every stage that were issued
        for (int st = 0; st < NST; ++st) {
            mbar_wait_drain(smem_addr(&sh.full_k[st]), 0, kWait / 64);
            mbar_wait_drain(smem_addr(&sh.full_k[st]), 1, kWait / 64);
            mbar_wait_drain(smem_addr(&sh.full_v[st]), 0, kWait / 64);
            mbar_wait_drain(smem_addr(&sh.full_v[st]), 1, kWait / 64);
        }
    }
}

// One query row of a unit that several CTAs took parts of: out = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c.
// The warps of the block take parts in turn, so a row of many parts is not one warp's chain.
constexpr int kMergeWarps = 4;
template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32) tree_merge_kernel(const TreeArgs a, int rows_tile) {
    const int rows_all = a.n_draft * a.group;
    const int row = blockIdx.x % rows_all, rt = row / rows_tile, r = row - rt * rows_tile;
    const int bg = blockIdx.x / rows_all, b = bg / a.pool.kv_heads, g = bg - b * a.pool.kv_heads;
    const int2 part = a.parts[bg * a.row_tiles + rt];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (part.x == part.y) return;
    __shared__ float s_m[kMergeWarps], s_l[kMergeWarps], s_o[kMergeWarps][D];
    constexpr int PER = (D + 31) / 32;
    float m = -INFINITY, l = 0.0f, o[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = 0.0f;
    for (int c = part.x + warp; c <= part.y; c += kMergeWarps) {
        const long long slot = (2ll * c + (c == part.x ? 1 : 0)) * rows_tile + r;
        const float2 ml = a.ws_ml[slot];
        float v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = lane + 32 * i < D ? a.ws_o[slot * D + lane + 32 * i] : 0.0f;
        const float mn = fmaxf(m, ml.x);
        if (mn == -INFINITY) continue;
        const float f = ex2(m - mn), h = ml.x == -INFINITY ? 0.0f : ex2(ml.x - mn);
        l = l * f + ml.y * h;
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] = o[i] * f + (h == 0.0f ? 0.0f : v[i] * h);
        m = mn;
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < D) s_o[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float mt = -INFINITY, lt = 0.0f;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) mt = fmaxf(mt, s_m[w]);
    float f[kMergeWarps];
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) {
        f[w] = s_m[w] == -INFINITY ? 0.0f : ex2(s_m[w] - mt);
        lt += s_l[w] * f[w];
    }
    const int t = row / a.group, hq = g * a.group + row - t * a.group;
    const long long at = ((long long)b * a.n_draft + t) * a.q_heads + hq;
    const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
    for (int d = threadIdx.x; d < D; d += kMergeWarps * 32) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) v += f[w] == 0.0f ? 0.0f : s_o[w][d] * f[w];
        v *= inv;
        if (a.out_dtype == EKV_DTYPE_F32) ((float *)a.out)[at * D + d] = v;
        else ((uint16_t *)a.out)[at * D + d] = f32_to_bf16_bits(v);
    }
    if (a.lse && threadIdx.x == 0) a.lse[at] = lt == 0.0f ? -INFINITY : (mt + __log2f(lt)) * 0.6931471805599453f;
}

// ---- host side ----
// Row tiles: 16 rows are one warp's registers (32 up to head_dim 128); more rows take four warps' rows, so
// that a tile of keys is read from shared memory once per 64 rows.
enum class Shape { R16, R32, R64 };

Shape shape_for(int head_dim, int rows) {
    if (rows <= 16) return Shape::R16;
    if (rows <= 32 && head_dim <= 128) return Shape::R32;
    return Shape::R64;
}
int tile_rows(Shape s) { return s == Shape::R16 ? 16 : s == Shape::R32 ? 32 : 64; }

int ctas_per_sm(Shape s, int head_dim) { return rows_ctas(head_dim, s == Shape::R32 ? 2 : 1); }

struct WsLayout {
    size_t parts, ml, o, total;
};
WsLayout ws_layout(const PoolView &p, int n_batch, int rows, int rt, int sms) {
    const Shape sh = shape_for(p.head_dim, rows);
    const size_t slots = 2ull * sms * ctas_per_sm(sh, p.head_dim) * tile_rows(sh);
    WsLayout w;
    w.parts = 0;
    w.ml = ((size_t)n_batch * p.kv_heads * rt * sizeof(int2) + 255) / 256 * 256;
    w.o = w.ml + slots * sizeof(float2);
    w.total = w.o + slots * p.head_dim * sizeof(float);
    return w;
}

template <int D, bool Q8, int MT, int WR, int WK>
int launch_rows(const TreeArgs &a, int grid, cudaStream_t s) {
    using C = Cfg<D, Q8, MT, WR, WK>;
    auto k = tree_rows_kernel<D, Q8, MT, WR, WK>;
    // the base is rounded up to 1024 bytes inside the kernel
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return EKV_ERR_CUDA;
    k<<<grid, C::THREADS, C::SMEM, s>>>(a);
    if (cudaGetLastError() != cudaSuccess) return EKV_ERR_CUDA;
    note_launches(1);
    return EKV_OK;
}

template <int D, bool Q8>
int launch_shape(const TreeArgs &a, Shape sh, int grid, cudaStream_t s) {
    switch (sh) {
        case Shape::R16: return launch_rows<D, Q8, 1, 1, 4>(a, grid, s);
        case Shape::R32:
            if constexpr (D <= 128) return launch_rows<D, Q8, 2, 1, 4>(a, grid, s);
            return EKV_ERR_UNSUPPORTED;
        default: return launch_rows<D, Q8, 1, 4, 1>(a, grid, s);
    }
}

template <int D>
int launch_dim(const TreeArgs &a, Shape sh, int grid, cudaStream_t s) {
    int rc;
    if (a.pool.dtype == EKV_DTYPE_Q8_0) {
        if constexpr (D % 32 == 0) rc = launch_shape<D, true>(a, sh, grid, s);
        else rc = EKV_ERR_UNSUPPORTED;
    } else {
        rc = launch_shape<D, false>(a, sh, grid, s);
    }
    if (rc || !a.split) return rc;
    const int rows = a.n_draft * a.group;
    tree_merge_kernel<D><<<a.n_batch * a.pool.kv_heads * rows, kMergeWarps * 32, 0, s>>>(a, tile_rows(sh));
    if (cudaGetLastError() != cudaSuccess) return EKV_ERR_CUDA;
    note_launches(1);
    return EKV_OK;
}

}  // namespace

size_t tree_workspace(const PoolView &p, int n_batch, int n_draft, int q_heads, int sms) {
    const int rows = n_draft * (q_heads / p.kv_heads);
    const int tr = tile_rows(shape_for(p.head_dim, rows));
    return ws_layout(p, n_batch, rows, (rows + tr - 1) / tr, sms).total;
}

int launch_tree_attention(TreeArgs a, int max_len, void *ws, size_t ws_bytes, int sms, cudaStream_t s) {
    const int rows = a.n_draft * a.group;
    const Shape sh = shape_for(a.pool.head_dim, rows);
    a.row_tiles = (rows + tile_rows(sh) - 1) / tile_rows(sh);
    const int64_t units = (int64_t)a.n_batch * a.pool.kv_heads * a.row_tiles;
    const int64_t all_rows = (int64_t)a.n_batch * a.pool.kv_heads * rows;
    if (units > INT32_MAX || all_rows > INT32_MAX) return EKV_ERR_INVALID_ARG;
    const WsLayout w = ws_layout(a.pool, a.n_batch, rows, a.row_tiles, sms);
    const int64_t unit_tiles = (max_len + kTile - 1) / kTile + 1;
    const int full = sms * ctas_per_sm(sh, a.pool.head_dim);
    // Units of one or two tiles are not worth a second launch; without a workspace a unit is one CTA's.
    a.split = ws != nullptr && ws_bytes >= w.total && unit_tiles > 2;
    int64_t grid = units;
    if (a.split) {
        grid = std::min<int64_t>(full, units * unit_tiles);
        a.parts = (int2 *)ws;
        a.ws_ml = (float2 *)((uint8_t *)ws + w.ml);
        a.ws_o = (float *)((uint8_t *)ws + w.o);
    }
    switch (a.pool.head_dim) {
        case 48: return launch_dim<48>(a, sh, (int)grid, s);
        case 64: return launch_dim<64>(a, sh, (int)grid, s);
        case 128: return launch_dim<128>(a, sh, (int)grid, s);
        case 256: return launch_dim<256>(a, sh, (int)grid, s);
        default: return EKV_ERR_UNSUPPORTED;
    }
}

}  // namespace ekv
