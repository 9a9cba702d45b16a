// ekv_tree.cu -- attention of a tree of drafted tokens over the paged cache (one token: plain decoding).
//
// For request b, drafted token t and query head h (KV head h / group), over the cached keys and those
// drafted keys that t's ancestor word names:
//   s_k = scale * q.k  (or cap * tanh(scale * q.k / cap)),  out = sum exp(s_k - m) v_k / sum exp(s_k - m),
//   lse = m + ln sum exp(s_k - m).
// For bf16 outputs over bf16 pages probabilities are rounded to bf16 for the products with V, and the output is divided by
// the sum of the rounded ones (a row with one heavy key would carry that key's rounding otherwise); lse takes the sum before
// rounding. For f32 outputs the probabilities, and over 8-bit pages p times the value's scale, a different number per 32
// columns, are two bf16 parts each, and the output is divided by the plain sum: off by 2^-16 of sum p |v| instead of 2^-8.
// The second parts cost 0 to 8% of an f32 call: 16 requests of 16 k keys 163.0 -> 163.2 us, 64 requests of 816 keys of 256
// columns 13.5 -> 14.6. 8-bit pages take them for bf16 outputs too: as one part, a heavy key's 32 columns were all off by up to
// 2^-8.
// One pass over the keys: a warp keeps the reference maximum m, the sum and the output of its rows in
// registers (the running softmax of Milakov and Gimelshein 2018, with the output as in flash attention,
// Dao et al. 2022). m moves only when a score is more than 2^8 above it; every quotient is exact about that.
//
// Products are taken transposed, S^T = K Q^T and O^T = V^T P^T: keys and value columns fill the 16 rows of
// the matrix instruction and query rows its 8 columns, so that the usual 4 or 8 rows of a decoded token's KV
// head waste nothing, and a row's output over D columns takes D / 4 registers of a thread for 8 rows.
// Bound and figures: with up to 16 rows of a KV head the bytes: 16 requests of 16 k keys, 8 KV heads of 128 columns in
// bf16 (976 MB), 4 rows each, take 151 us, 6.5 TB/s, 99% of the measured copy rate. Short caches are bound by the chain
// launch, lengths, block ids, first tile, a few tiles, join: one token over 816 keys 8.4 us, 64 requests of 816 Q8_0 keys
// 20 us where their bytes take 4.1. More rows are bound by the matrix instructions of one or two warps per
// scheduler, and are the tile kernel's but for Q8_0 at head_dim 256, head_dim 48 and some capped calls.
#include <algorithm>

#include "ekv_decode.cuh"

namespace ekv {
namespace {

using namespace decode;
using namespace sm100;


// CTAs per SM: two where a thread's share of the output (8 * NR rows by D columns over a warp) leaves the
// registers for it and two tiles in flight fit the shared memory of half an SM.
constexpr int rows_ctas(int d, bool q8, int nr, int wr) {
    return d * nr > 256 || wr * 8 * nr > 64 || (d > 128 && !q8) || (d > 128 && wr > 1) ? 1 : 2;
}

constexpr int kMaxCluster = 8;

// WR row groups of 8 * NR rows times WK groups of 64 / WK keys: one warp each, and one feeder warp.
template <int D, bool Q8, int NR, int WR, int WK>
struct Cfg {
    using T = TileCfg<D, Q8>;
    static constexpr int NW = WR * WK, NC = NW * 32, THREADS = NC + 32;
    static constexpr int ROWS = 8 * NR * WR;
    static constexpr int KPW = kTile / WK;          // keys of a tile per warp
    static constexpr int NB = KPW / 16;             // 16-key steps per warp and tile
    // drafted keys per tile: bf16 rows in the tile's own layout, or padded rows where the tile is Q8_0
    static constexpr int DT = Q8 ? 32 : kTile;
    static constexpr int DROW = 2 * D + 16;         // bytes of a drafted row in a Q8_0 kernel
    static constexpr int STAGE_MIN = 2 * T::KV_BYTES, STAGE_DRAFT = Q8 ? 2 * DT * DROW : 0;
    static constexpr int STAGE = ((STAGE_MIN > STAGE_DRAFT ? STAGE_MIN : STAGE_DRAFT) + 1023) / 1024 * 1024;
    static constexpr int V_OFF = T::KV_BYTES, DRAFT_V_OFF = Q8 ? DT * DROW : T::KV_BYTES;
    // columns that the key groups' outputs are joined in at a time: 16 KB of rows (or all columns)
    static constexpr int X_FIT = WK * ROWS <= 32 ? 128 : WK * ROWS <= 64 ? 64 : 32;
    static constexpr int X_COLS = X_FIT < D ? X_FIT : D <= 32 ? 32 : D <= 64 ? 64 : 128;
    static constexpr int X_BYTES = WK * ROWS * X_COLS * 4;
    static constexpr int ML_BYTES = WK * ROWS * 16;
    // query rows in shared memory where the output's share of the registers leaves no room for them
    static constexpr bool Q_SMEM = D * NR > 256;
    static constexpr int Q_BYTES = Q_SMEM ? ROWS * q_row_bytes<D, Q8>() : 0;
    // what the CTAs of a cluster send one another: this CTA's share of the unit's outputs and all rows' maxima and
    // sums, from each of them (few rows only: a large unit is better split)
    static constexpr bool CLUSTERS = ROWS * D <= 2048;
    static constexpr int P_BYTES = CLUSTERS ? ROWS * D * 4 + kMaxCluster * (ROWS + 1) * 16 : 0;
    static constexpr int FIXED = X_BYTES + ML_BYTES + Q_BYTES + P_BYTES + 1024 + 1024;
    static constexpr int CTAS = rows_ctas(D, Q8, NR, WR);
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
    int table[kTableWindow];
};

// Column of output accumulator (16-column step ds, element i) of lane row kq. Q8_0 kernels take the columns of a
// 32-column group in the order that one word of a key's row gives them to a lane.
template <bool Q8>
__device__ __forceinline__ int o_col(int ds, int kq, int i) {
    return Q8 ? 32 * (ds >> 1) + 4 * kq + 2 * (ds & 1) + (i >> 1) : 16 * ds + kq + 8 * (i >> 1);
}

// FINE (f32 outputs): probabilities as two bf16 parts for the products with V, over 8-bit pages always.
template <int D, bool Q8, bool FINE, int NR, int WR, int WK>
__global__ void __launch_bounds__(Cfg<D, Q8, NR, WR, WK>::THREADS, Cfg<D, Q8, NR, WR, WK>::CTAS)
    tree_rows_kernel(const TreeArgs a) {
    using C = Cfg<D, Q8, NR, WR, WK>;
    static_assert(FINE || !Q8, "8-bit pages have one form");
    constexpr int NST = C::NST, KS = D / 16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float *xb = (float *)(smem + NST * C::STAGE);                   // [WK][ROWS][kXCols]
    float4 *sml = (float4 *)(smem + NST * C::STAGE + C::X_BYTES);   // [WK][ROWS]: maximum, sum, rounded sum
    using Sh = Shared<NST>;
    static_assert(sizeof(Sh) <= 1024, "barrier block");
    Sh &sh = *(Sh *)(smem + NST * C::STAGE + C::X_BYTES + C::ML_BYTES);
    uint8_t *sq = smem + NST * C::STAGE + C::X_BYTES + C::ML_BYTES + 1024;  // [ROWS] query rows (Q_SMEM)
    float4 *part_o = (float4 *)(sq + C::Q_BYTES);                       // [cluster][its share of the unit's float4 outputs]
    float4 *part_ml = part_o + C::ROWS * D / 4 + kMaxCluster;           // [cluster][ROWS]
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
    // without the split a cluster of CTAs takes one unit's tiles in equal parts and joins its outputs through their
    // shared memory
    const int unit = blockIdx.x / a.cluster, rank = blockIdx.x - unit * a.cluster;
    if (C::CLUSTERS && a.cluster > 1) cluster_arrive_relaxed();  // (waited for before anything is sent)
    Range rg;
    grid_wait();
    grid_launch_next();  // the merge's blocks may take their places; they wait for this grid's end
    if (a.split) {
        rg = find_range<C::THREADS>(a.n_batch, units_per_req, sh.range,
                                    [&](int b) { return load_req(a, b, blockIdx.x == 0); }, unit_tiles);
    } else {
        __syncthreads();
        rg.b = unit / units_per_req;
        rg.req = load_req(a, rg.b, threadIdx.x == 0 && rank == 0);
        rg.base = rg.lo = rg.hi = rg.total = 0;
        rg.ctas = 0;
    }

    int st = 0, turn = 0;  // stage of the next tile, and how often the ring went round
    auto advance = [&]() {
        if (++st == NST) {
            st = 0;
            ++turn;
        }
    };
    bool ok = true;
    TableWindow tw;  // (the feeder's)
    tw.reset(sh.table);
    int b = rg.b;
    uint32_t base = rg.base;
    Req rq = rg.req;
    int rq_of = b;  // the request that rq describes
    for (uint32_t x = rg.lo; (x < rg.hi || !a.split) && b < a.n_batch;) {
        if (b != rq_of) rq = load_req(a, b, false), rq_of = b;
        const int n_tiles = unit_tiles(rq);
        const uint32_t span = (uint32_t)n_tiles * units_per_req;
        if (a.split && x >= base + span) {
            base += span;
            ++b;
            continue;
        }
        const int u = a.split ? (int)((x - base) / (uint32_t)n_tiles) : unit - b * units_per_req;
        const int t0 = a.split ? (int)(x - base) - u * n_tiles : rank * n_tiles / a.cluster;
        const int t1 = a.split ? min(n_tiles, t0 + (int)(rg.hi - x)) : (rank + 1) * n_tiles / a.cluster;
        const int g = u / a.row_tiles, row0 = (u - g * a.row_tiles) * C::ROWS;
        const int rows = min(C::ROWS, rows_all - row0);
        const int p_tiles = (rq.n_prefix + kTile - 1) / kTile;
        const long long kv_row = ((long long)b * a.n_draft * hk + g) * D;  // drafted token 0 of this head
        // query row r of the unit, or null where it does not take part
        auto q_row = [&](int r) -> const uint16_t * {
            const int t = row_token(a, r);
            if (r >= rows_all || t >= rq.n_nodes) return nullptr;
            return a.q + (((long long)b * a.n_draft + t) * a.q_heads + g * a.group + (r - t * a.group)) * D;
        };

        if (warp == C::NW) {
            // ---- feeder ----
            Piece next = find_piece<D, Q8>(a, rq, g, t0 * kTile, tw, lane);
            if (a.split && lane == 0 && t0 == 0) {  // the CTAs of this unit: tile x is CTA ((x + 1) G - 1) / T's
                const unsigned long long end = base + (uint32_t)(u + 1) * n_tiles;
                a.parts[b * units_per_req + u] = make_int2(blockIdx.x, (int)((end * rg.ctas - 1) / rg.total));
            }
            for (int j = t0; j < t1; ++j, advance()) {
                const Piece pc = next;
                if (j + 1 < min(t1, p_tiles)) next = find_piece<D, Q8>(a, rq, g, (j + 1) * kTile, tw, lane);
                if (turn > 0) ok = ok && warp_wait(smem_addr(&sh.empty[st]), (turn - 1) & 1, abort);
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
            const int kq = lane >> 2, c = lane & 3;  // key (or value column) and query row pair of the lane's elements
            const int wrow = wr * 8 * NR;
            // query operands: row wrow + 8 n + kq
            uint32_t qf[C::Q_SMEM ? 1 : NR][C::Q_SMEM ? 1 : KS][2];
            int t_of[NR][2];  // drafted token of rows wrow + 8 n + 2 c (+ 1), -1 where the row does not take part
#pragma unroll
            for (int n = 0; n < NR; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = row0 + wrow + 8 * n + 2 * c + e, t = row_token(a, r);
                    t_of[n][e] = r < rows_all && t < rq.n_nodes ? t : -1;
                }
                if constexpr (!C::Q_SMEM) {
                    const uint16_t *src = q_row(row0 + wrow + 8 * n + kq);
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int half = 0; half < 2; ++half)
                            qf[n][ks][half] = src ? __ldg((const uint32_t *)(src + q_col<Q8>(ks, c, half))) : 0u;
                }
            }
            if constexpr (C::Q_SMEM) {  // the last rows were done with at the barriers of their end
                stage_q_rows<D, Q8>(smem_addr(sq), C::ROWS, a.q, warp, C::NW, lane, [&](int r) { return q_row(row0 + r); });
                cp_async_wait_all();
                asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
            }
            // operands of steps 2 i and 2 i + 1 (D is a multiple of 32 where they come from shared memory)
            auto load_q2 = [&](int n, int i, uint32_t (&f)[4]) {
                if constexpr (C::Q_SMEM) {
                    load_q_steps<D, Q8>(smem_addr(sq) + (wrow + 8 * n) * q_row_bytes<D, Q8>(), i, lane, f);
                } else {
                    f[0] = qf[n][2 * i][0];
                    f[1] = qf[n][2 * i][1];
                    if (2 * i + 1 < KS) {
                        f[2] = qf[n][2 * i + 1][0];
                        f[3] = qf[n][2 * i + 1][1];
                    }
                }
            };
            float o[NR][KS][4];  // O^T: columns o_col(ds, kq, i), row 2 c + (i & 1)
            float mx[NR][2], sum[NR][2], rsum[NR][2];
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                mx[n][0] = mx[n][1] = -INFINITY;
                sum[n][0] = sum[n][1] = rsum[n][0] = rsum[n][1] = 0.0f;
#pragma unroll
                for (int ds = 0; ds < KS; ++ds)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[n][ds][i] = 0.0f;
            }
            const ScoreFn score{a.scale_log2, a.cap_log2, a.cap_in};

            for (int j = t0; j < t1; ++j, advance()) {
                const int par = turn & 1;
                uint8_t *tile = smem + st * C::STAGE;
                const uint32_t sk = smem_addr(tile);
                const bool draft = j >= p_tiles;
                const int d0 = (j - p_tiles) * C::DT;
                const int valid = draft ? min(C::DT, rq.n_nodes - d0) : min(kTile, rq.n_prefix - j * kTile);
                const uint32_t sv = sk + (draft ? C::DRAFT_V_OFF : C::V_OFF);
                ok = ok && warp_wait(smem_addr(&sh.full_k[st]), par, abort);
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                bool v_ready = false;
#pragma unroll 1
                for (int kb = 0; kb < C::NB; ++kb) {
                    const int key0 = wk * C::KPW + kb * 16;  // 16 keys of the tile
                    if (key0 >= valid) break;
                    // ---- S^T = K Q^T: keys kq, kq + 8; rows 2 c, 2 c + 1 ----
                    float s[NR][4];
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
                    if constexpr (!Q8) {
#pragma unroll
                        for (int i = 0; i < (KS + 1) / 2; ++i) {
                            uint32_t k0[4], k1[4];
                            load_k_rows<D>(sk, key0, 2 * i, lane, k0);
                            if (2 * i + 1 < KS) load_k_rows<D>(sk, key0, 2 * i + 1, lane, k1);
#pragma unroll
                            for (int n = 0; n < NR; ++n) {
                                uint32_t f[4];
                                load_q2(n, i, f);
                                mma_bf16(s[n], k0, f[0], f[1]);
                                if (2 * i + 1 < KS) mma_bf16(s[n], k1, f[2], f[3]);
                            }
                        }
                    } else if (draft) {
#pragma unroll
                        for (int i = 0; i < KS / 2; ++i) {
                            // 8 columns of two keys in one load: steps 2 i and 2 i + 1
                            const uint32_t at = sk + (key0 + kq) * C::DROW + 2 * (32 * i + 8 * c);
                            const uint4 w0 = lds128(at), w1 = lds128(at + 8 * C::DROW);
                            const uint32_t k0[4] = {w0.x, w1.x, w0.y, w1.y}, k1[4] = {w0.z, w1.z, w0.w, w1.w};
#pragma unroll
                            for (int n = 0; n < NR; ++n) {
                                uint32_t f[4];
                                load_q2(n, i, f);
                                mma_bf16(s[n], k0, f[0], f[1]);
                                mma_bf16(s[n], k1, f[2], f[3]);
                            }
                        }
                    } else {
                        // integer products of a 32-column group are exact; the keys' scales join in f32
                        using T = TileCfg<D, true>;
                        uint32_t sc0[(T::G32 + 1) / 2], sc1[(T::G32 + 1) / 2];
                        load_scales<T::G32>(sk + T::SCALES + (key0 + kq) * T::G32 * 2, sc0);
                        load_scales<T::G32>(sk + T::SCALES + (key0 + kq + 8) * T::G32 * 2, sc1);
#pragma unroll
                        for (int gr = 0; gr < T::G32; ++gr) {
                            const uint2 w0 = lds64(sk + q8_qs_off(key0 + kq, 32 * gr + 8 * c, D));
                            const uint2 w1 = lds64(sk + q8_qs_off(key0 + kq + 8, 32 * gr + 8 * c, D));
                            uint32_t k0[4], k1[4];
                            int8x4_to_bf16(w0.x, k0[0], k0[2]);
                            int8x4_to_bf16(w1.x, k0[1], k0[3]);
                            int8x4_to_bf16(w0.y, k1[0], k1[2]);
                            int8x4_to_bf16(w1.y, k1[1], k1[3]);
                            const float f0 = scale_of(sc0, gr), f1 = scale_of(sc1, gr);
#pragma unroll
                            for (int n = 0; n < NR; ++n) {
                                uint32_t f[4];
                                load_q2(n, gr, f);
                                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                mma_bf16(acc, k0, f[0], f[1]);
                                mma_bf16(acc, k1, f[2], f[3]);
                                s[n][0] = fmaf(acc[0], f0, s[n][0]);
                                s[n][1] = fmaf(acc[1], f0, s[n][1]);
                                s[n][2] = fmaf(acc[2], f1, s[n][2]);
                                s[n][3] = fmaf(acc[3], f1, s[n][3]);
                            }
                        }
                    }
                    // ---- mask, reference maximum, exponentials ----
                    const bool masked = draft || key0 + 16 > valid;
                    uint32_t vis[NR][2];  // draft tiles: bit k, key0 + k visible to the row
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            vis[n][e] = 0xffffu;
                            if (masked) {
                                uint64_t w = valid >= 64 ? ~0ull : (1ull << valid) - 1;
                                if (draft) {
                                    const int t = t_of[n][e];
                                    w &= t < 0 ? 0ull
                                         : a.ancestors ? __ldg(a.ancestors + (long long)b * a.n_draft + t) >> d0
                                                       : (t >= 63 ? ~0ull : (2ull << t) - 1) >> d0;
                                }
                                vis[n][e] = (uint32_t)(w >> key0) & 0xffffu;
                            }
                        }
                    bool above = false;
                    score(*(float(*)[4 * NR])s);
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (masked && !((vis[n][i & 1] >> (kq + 8 * (i >> 1))) & 1u)) s[n][i] = -INFINITY;
                        }
                        above = above || fmaxf(s[n][0], s[n][2]) > mx[n][0] + 8.0f || fmaxf(s[n][1], s[n][3]) > mx[n][1] + 8.0f;
                    }
                    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                        for (int n = 0; n < NR; ++n) {
                            float f[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float m = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
                                for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
                                m = fmaxf(m, mx[n][e]);
                                f[e] = m == -INFINITY ? 1.0f : ex2(mx[n][e] - m);
                                mx[n][e] = m;
                                sum[n][e] *= f[e];
                                rsum[n][e] *= f[e];
                            }
#pragma unroll
                            for (int ds = 0; ds < KS; ++ds)
#pragma unroll
                                for (int i = 0; i < 4; ++i) o[n][ds][i] *= f[i & 1];
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        const float u0 = mx[n][0] == -INFINITY ? 0.0f : mx[n][0], u1 = mx[n][1] == -INFINITY ? 0.0f : mx[n][1];
                        s[n][0] = ex2(s[n][0] - u0);
                        s[n][1] = ex2(s[n][1] - u1);
                        s[n][2] = ex2(s[n][2] - u0);
                        s[n][3] = ex2(s[n][3] - u1);
                        sum[n][0] += s[n][0] + s[n][2];
                        sum[n][1] += s[n][1] + s[n][3];
                    }
                    // ---- O^T += V^T P^T ----
                    if (!v_ready) {
                        ok = warp_wait(smem_addr(&sh.full_v[st]), par, abort);
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
                        uint32_t p[NR][2], pl[FINE ? NR : 1][2];  // P^T, and what its rounding left
#pragma unroll
                        for (int n = 0; n < NR; ++n) {
                            const uint32_t w0 = pack_bf16(s[n][0], s[n][1]), w1 = pack_bf16(s[n][2], s[n][3]);
                            const float h[4] = {__uint_as_float(w0 << 16), __uint_as_float(w0 & 0xffff0000u), __uint_as_float(w1 << 16),
                                                __uint_as_float(w1 & 0xffff0000u)};
                            if constexpr (FINE) {
                                pl[n][0] = movmatrix_trans(pack_bf16(s[n][0] - h[0], s[n][1] - h[1]));
                                pl[n][1] = movmatrix_trans(pack_bf16(s[n][2] - h[2], s[n][3] - h[3]));
                            } else {
                                rsum[n][0] += h[0] + h[2];
                                rsum[n][1] += h[1] + h[3];
                            }
                            p[n][0] = movmatrix_trans(w0);
                            p[n][1] = movmatrix_trans(w1);
                        }
#pragma unroll
                        for (int ds = 0; ds < KS; ++ds) {
                            uint32_t vf[4];
                            load_v_cols<D>(sv, key0, ds, lane, vf);
#pragma unroll
                            for (int n = 0; n < NR; ++n) mma_bf16(o[n][ds], vf, p[n][0], p[n][1]);
                            if constexpr (FINE) {
#pragma unroll
                                for (int n = 0; n < NR; ++n) mma_bf16(o[n][ds], vf, pl[n][0], pl[n][1]);
                            }
                        }
                    } else {
                        constexpr int G = D / 32;
                        const int kr[4] = {key0 + 2 * c, key0 + 2 * c + 1, key0 + 2 * c + 8, key0 + 2 * c + 9};
                        uint32_t sc[4][(G + 1) / 2];
                        if (!draft)
#pragma unroll
                            for (int k = 0; k < 4; ++k) load_scales<G>(sv + TileCfg<D, Q8>::SCALES + kr[k] * G * 2, sc[k]);
                        // the probabilities of row kq and keys kr, from the keys' lanes: as two bf16 each, which hold
                        // 16 bits of them, through the 16-bit transpose
                        float pt[NR][4];
#pragma unroll
                        for (int n = 0; n < NR; ++n) {
                            const uint32_t h0 = pack_bf16(s[n][0], s[n][1]), h1 = pack_bf16(s[n][2], s[n][3]);
                            const uint32_t l0 = pack_bf16(s[n][0] - __uint_as_float(h0 << 16), s[n][1] - __uint_as_float(h0 & 0xffff0000u));
                            const uint32_t l1 = pack_bf16(s[n][2] - __uint_as_float(h1 << 16), s[n][3] - __uint_as_float(h1 & 0xffff0000u));
                            const uint32_t a0 = movmatrix_trans(h0), a1 = movmatrix_trans(h1), b0 = movmatrix_trans(l0), b1 = movmatrix_trans(l1);
                            pt[n][0] = __uint_as_float(a0 << 16) + __uint_as_float(b0 << 16);
                            pt[n][1] = __uint_as_float(a0 & 0xffff0000u) + __uint_as_float(b0 & 0xffff0000u);
                            pt[n][2] = __uint_as_float(a1 << 16) + __uint_as_float(b1 << 16);
                            pt[n][3] = __uint_as_float(a1 & 0xffff0000u) + __uint_as_float(b1 & 0xffff0000u);
                        }
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) {
                            uint32_t v0[4], v1[4];  // operands of the group's two 16-column steps
                            float f[4] = {1.0f, 1.0f, 1.0f, 1.0f};
                            if (draft) {
                                uint2 w[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) w[k] = lds64(sv + kr[k] * C::DROW + (32 * gr + 4 * kq) * 2);
                                v0[0] = __byte_perm(w[0].x, w[1].x, 0x5410);
                                v0[1] = __byte_perm(w[0].x, w[1].x, 0x7632);
                                v0[2] = __byte_perm(w[2].x, w[3].x, 0x5410);
                                v0[3] = __byte_perm(w[2].x, w[3].x, 0x7632);
                                v1[0] = __byte_perm(w[0].y, w[1].y, 0x5410);
                                v1[1] = __byte_perm(w[0].y, w[1].y, 0x7632);
                                v1[2] = __byte_perm(w[2].y, w[3].y, 0x5410);
                                v1[3] = __byte_perm(w[2].y, w[3].y, 0x7632);
                            } else {
                                uint32_t w[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) w[k] = lds32(sv + q8_qs_off(kr[k], 32 * gr + 4 * kq, D));
                                int8x4_to_bf16(__byte_perm(w[0], w[1], 0x5140), v0[0], v0[1]);
                                int8x4_to_bf16(__byte_perm(w[2], w[3], 0x5140), v0[2], v0[3]);
                                int8x4_to_bf16(__byte_perm(w[0], w[1], 0x7362), v1[0], v1[1]);
                                int8x4_to_bf16(__byte_perm(w[2], w[3], 0x7362), v1[2], v1[3]);
#pragma unroll
                                for (int k = 0; k < 4; ++k) f[k] = scale_of(sc[k], gr);
                            }
                            // The values' scales ride on the probabilities, as two bf16 parts: one part would put a whole
                            // group of 32 columns off by the same 2^-8. An infinite scale has no remainder (inf - inf), and
                            // any finite number serves for it. The second part's products cost 3 to 10% of a call: 64 requests
                            // of 816 keys, 256 columns, 8 rows 18.9 -> 19.8 us, 512 rows 557 -> 612.
#pragma unroll
                            for (int n = 0; n < NR; ++n) {
                                const uint64_t x01 = fma_pair(pair_of(pt[n][0], pt[n][1]), pair_of(f[0], f[1]), 0);
                                const uint64_t x23 = fma_pair(pair_of(pt[n][2], pt[n][3]), pair_of(f[2], f[3]), 0);
                                const uint32_t p0 = pack_bf16(of_pair(x01).x, of_pair(x01).y), p1 = pack_bf16(of_pair(x23).x, of_pair(x23).y);
                                const uint64_t minus = pair_of(-1.0f, -1.0f);
                                const float2 d0 = of_pair(fma_pair(pair_of(__uint_as_float(p0 << 16), __uint_as_float(p0 & 0xffff0000u)), minus, x01));
                                const float2 d1 = of_pair(fma_pair(pair_of(__uint_as_float(p1 << 16), __uint_as_float(p1 & 0xffff0000u)), minus, x23));
                                const float r[4] = {fminf(d0.x, 3e38f), fminf(d0.y, 3e38f), fminf(d1.x, 3e38f), fminf(d1.y, 3e38f)};
                                const uint32_t r0 = pack_bf16(r[0], r[1]), r1 = pack_bf16(r[2], r[3]);
                                mma_bf16(o[n][2 * gr], v0, p0, p1);
                                mma_bf16(o[n][2 * gr + 1], v1, p0, p1);
                                mma_bf16(o[n][2 * gr], v0, r0, r1);
                                mma_bf16(o[n][2 * gr + 1], v1, r0, r1);
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
                            for (int n = 0; n < NR; ++n) {
                                float pk[2];
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    pk[e] = __shfl_sync(0xffffffffu, k < 8 ? s[n][e] : s[n][e + 2], (k & 7) * 4 + c);
#pragma unroll
                                for (int ds = 0; ds < KS; ++ds)
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        const float y = bf16_bits_to_f32(__ldg(v + o_col<Q8>(ds, kq, i)));
                                        if (!isfinite(y) && ((vis[n][i & 1] >> k) & 1u)) o[n][ds][i] = fmaf(pk[i & 1], y, o[n][ds][i]);
                                    }
                            }
                        }
                    }
                }
                if (ok && !v_ready) {  // no key of this tile is the warp's: still stay in step with the stage
                    ok = warp_wait(smem_addr(&sh.full_v[st]), par, abort);
                    if (!ok) *abort = 1;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&sh.empty[st]));
            }

            // ---- join the key groups, write the rows ----
            if (C::CLUSTERS && a.cluster > 1) {  // the other CTAs have started
                __syncwarp();
                cluster_wait();
            }
            float scale_o[NR][2];
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float l = sum[n][e], lr = FINE ? sum[n][e] : rsum[n][e];
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) {
                        l += __shfl_xor_sync(0xffffffffu, l, x);
                        lr += __shfl_xor_sync(0xffffffffu, lr, x);
                    }
                    if (kq == 0) sml[wk * C::ROWS + wrow + 8 * n + 2 * c + e] = make_float4(mx[n][e], l, lr, 0.0f);
                }
            asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
            const bool joins = C::CLUSTERS && a.cluster > 1, whole = t0 == 0 && t1 == n_tiles && !joins;
            const long long slot = 2ll * blockIdx.x + (t0 == 0 ? 1 : 0);
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = wrow + 8 * n + 2 * c + e;
                    float mt = -INFINITY, lt = 0.0f, lr = 0.0f;
#pragma unroll
                    for (int w = 0; w < WK; ++w) mt = fmaxf(mt, sml[w * C::ROWS + r].x);
                    const float mu = mt == -INFINITY ? 0.0f : mt;
#pragma unroll
                    for (int w = 0; w < WK; ++w) {
                        const float4 ml = sml[w * C::ROWS + r];
                        const float f = ex2(ml.x - mu);
                        lt += ml.y * f;
                        lr += ml.z * f;
                    }
                    scale_o[n][e] = mx[n][e] == -INFINITY ? 0.0f : ex2(mx[n][e] - mu);
                    if (whole) scale_o[n][e] = lr == 0.0f ? 0.0f : scale_o[n][e] / lr;
                    if (wk != 0 || kq != 0 || r >= rows) continue;
                    const bool off = t_of[n][e] < 0;
                    if (joins) {
                        const uint32_t at = smem_addr(part_ml + rank * C::ROWS + r);
                        for (int k = 0; k < a.cluster; ++k)
                            stc128(mapa_shared(at, k), off ? make_float4(-INFINITY, 0.0f, 0.0f, 0.0f) : make_float4(mt, lt, lr, 0.0f));
                    } else if (!whole) {
                        a.ws_ml[slot * C::ROWS + r] = off ? make_float4(-INFINITY, 0.0f, 0.0f, 0.0f) : make_float4(mt, lt, lr, 0.0f);
                    } else if (a.lse) {
                        const int t = row_token(a, row0 + r), hq = g * a.group + (row0 + r) - t * a.group;
                        a.lse[((long long)b * a.n_draft + t) * a.q_heads + hq] =
                            off || lt == 0.0f ? -INFINITY : (mt + __log2f(lt)) * 0.6931471805599453f;
                    }
                }
            const int share = (rows * (D / 4) + a.cluster - 1) / a.cluster;  // float4 outputs that a CTA of the cluster writes
            constexpr int XC = C::X_COLS, ROUNDS = (D + XC - 1) / XC;
#pragma unroll
            for (int cc = 0; cc < ROUNDS; ++cc) {
                constexpr int q4_max = XC / 4;
                const int q4 = min(XC, D - cc * XC) / 4;
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int d2 = 0; d2 < XC / 16; ++d2) {
                        const int ds = cc * (XC / 16) + d2;
                        if (ds >= KS) continue;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = wrow + 8 * n + 2 * c + (i & 1);
                            const int col = o_col<Q8>(ds, kq, i) - cc * XC;
                            // a warp without a key for the row has nothing (not 0 * its garbage)
                            const float f = scale_o[n][i & 1];
                            xb[(wk * C::ROWS + r) * XC + ((col + 4 * r) & (XC - 1))] = f == 0.0f ? 0.0f : o[n][ds][i] * f;
                        }
                    }
                asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
                for (int i = threadIdx.x; i < rows * q4; i += C::NC) {
                    const int r = q4 == q4_max ? i / q4_max : i / q4, col = (i - r * q4) * 4;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < WK; ++w) {
                        const float4 y = *(const float4 *)&xb[(w * C::ROWS + r) * XC + ((col + 4 * r) & (XC - 1))];
                        v.x += y.x;
                        v.y += y.y;
                        v.z += y.z;
                        v.w += y.w;
                    }
                    if (joins) {  // to the CTA that writes it
                        const int item = r * (D / 4) + (cc * XC + col) / 4, to = item / share;
                        stc128(mapa_shared(smem_addr(part_o + rank * share + item - to * share), to), v);
                        continue;
                    }
                    if (!whole) {
                        *(float4 *)(a.ws_o + (slot * C::ROWS + r) * D + cc * XC + col) = v;
                        continue;
                    }
                    const int t = row_token(a, row0 + r), hq = g * a.group + (row0 + r) - t * a.group;
                    if (t >= rq.n_nodes) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    const long long dst = (((long long)b * a.n_draft + t) * a.q_heads + hq) * D + cc * XC + col;
                    if (a.out_dtype == EKV_DTYPE_F32)
                        *(float4 *)((float *)a.out + dst) = v;
                    else
                        *(uint2 *)((uint16_t *)a.out + dst) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
                }
                // (the next unit's end has a barrier before these are written again)
                if (cc + 1 < ROUNDS) asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
            }
        }
        if constexpr (C::CLUSTERS)
            if (a.cluster > 1) {
                // out = sum_k 2^(m_k - m) o_k / sum_k 2^(m_k - m) l_k over the cluster's CTAs k
                __syncwarp();
                if (warp == C::NW) cluster_wait();
                cluster_sync();  // everyone's parts are here
                const int share = (rows * (D / 4) + a.cluster - 1) / a.cluster;
                for (int i = threadIdx.x; i < share && rank * share + i < rows * (D / 4); i += C::THREADS) {
                    const int item = rank * share + i, r = item / (D / 4), col = (item - r * (D / 4)) * 4;
                    float m = -INFINITY, l = 0.0f, lr = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int k = 0; k < a.cluster; ++k) m = fmaxf(m, part_ml[k * C::ROWS + r].x);
                    for (int k = 0; k < a.cluster; ++k) {
                        const float4 ml = part_ml[k * C::ROWS + r], y = part_o[k * share + i];
                        const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m);
                        l += f * ml.y;
                        lr += f * ml.z;
                        if (f == 0.0f) continue;  // (a part that saw nothing for the row)
                        v.x = fmaf(y.x, f, v.x);
                        v.y = fmaf(y.y, f, v.y);
                        v.z = fmaf(y.z, f, v.z);
                        v.w = fmaf(y.w, f, v.w);
                    }
                    const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
                    v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                    const int t = row_token(a, row0 + r), hq = g * a.group + (row0 + r) - t * a.group;
                    const long long at = ((long long)b * a.n_draft + t) * a.q_heads + hq;
                    if (a.out_dtype == EKV_DTYPE_F32) *(float4 *)((float *)a.out + at * D + col) = v;
                    else *(uint2 *)((uint16_t *)a.out + at * D + col) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
                    if (a.lse && col == 0) a.lse[at] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
                }
            }
        if (!a.split) break;
        x += t1 - t0;
    }
    if (!ok && lane == 0) report_error(a.pool.status, DEV_ERR_TIMEOUT, blockIdx.x, warp, 7);
    if (warp == C::NW && !ok && lane == 0) {
        // leave no copy writing this CTA's shared memory: the last uses of every stage that were issued
        for (int i = 0; i < NST; ++i) {
            mbar_wait_drain(smem_addr(&sh.full_k[i]), 0, kWait / 64);
            mbar_wait_drain(smem_addr(&sh.full_k[i]), 1, kWait / 64);
            mbar_wait_drain(smem_addr(&sh.full_v[i]), 0, kWait / 64);
            mbar_wait_drain(smem_addr(&sh.full_v[i]), 1, kWait / 64);
        }
    }
}

// Rows of units that several CTAs took parts of: out = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c. Two forms: a
// warp for four rows, whose parts are the same, so that 8 rows of parts are on their way at a time; or, where that
// leaves SMs empty, a block for one row, its warps taking parts in turn.
constexpr int kMergeWarps = 8, kMergeRows = 4;

struct MergeRow {  // one of a group's rows: where its result goes, and its parts
    int bg, rt, r;
    long long at;
};
__device__ __forceinline__ MergeRow merge_row(const TreeArgs &a, int bg, int row, int rows_tile) {
    MergeRow m;
    m.bg = bg;
    m.rt = row / rows_tile;
    m.r = row - m.rt * rows_tile;
    const int b = bg / a.pool.kv_heads, g = bg - b * a.pool.kv_heads, t = row_token(a, row);
    m.at = ((long long)b * a.n_draft + t) * a.q_heads + g * a.group + row - t * a.group;
    return m;
}
template <int D>
__device__ __forceinline__ void merge_put(const TreeArgs &a, long long at, int i, float4 v, float inv) {
    v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    if (a.out_dtype == EKV_DTYPE_F32) ((float4 *)((float *)a.out + at * D))[i] = v;
    else ((uint2 *)((uint16_t *)a.out + at * D))[i] = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}
__device__ __forceinline__ void merge_add(float4 &o, const float4 &v, float f) {
    if (f == 0.0f) return;  // (a part that saw nothing for the row: its output may be anything)
    o.x = fmaf(v.x, f, o.x);
    o.y = fmaf(v.y, f, o.y);
    o.z = fmaf(v.z, f, o.z);
    o.w = fmaf(v.w, f, o.w);
}

// Part c of row r of a unit whose first CTA is `first`.
__device__ __forceinline__ long long part_row(int c, int first, int rows_tile, int r) {
    return (2ll * c + (c == first ? 1 : 0)) * rows_tile + r;
}

template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32) tree_merge_rows_kernel(const TreeArgs a, int rows_tile, int n_groups) {
    constexpr int R = kMergeRows, PARTS = 32 / R, PER = (D + 127) / 128;  // float4 of a lane
    const int lane = threadIdx.x & 31, id = blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
    if (id >= n_groups) return;
    const int rows_all = a.n_draft * a.group, groups = (rows_all + R - 1) / R;
    const int bg = id / groups, row0 = (id - bg * groups) * R, rows = min(R, rows_all - row0);
    const int sub = min(lane % R, rows - 1);  // (rows of a group are in one row tile: its size is a multiple of 8)
    const MergeRow mine = merge_row(a, bg, row0 + sub, rows_tile);
    const int r0 = mine.r - sub;
    grid_wait();
    const int2 part = a.parts[bg * a.row_tiles + mine.rt];
    if (part.x == part.y) return;
    float m = -INFINITY;
    for (int c = part.x + lane / R; c <= part.y; c += PARTS) m = fmaxf(m, a.ws_ml[part_row(c, part.x, rows_tile, mine.r)].x);
#pragma unroll
    for (int x = R; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    float l = 0.0f, lr = 0.0f;
    float4 o[R][PER];
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
        for (int i = 0; i < PER; ++i) o[k][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c0 = part.x; c0 <= part.y; c0 += PARTS) {
        float f = 0.0f;
        const int c = c0 + lane / R;
        if (c <= part.y) {
            const float4 ml = a.ws_ml[part_row(c, part.x, rows_tile, mine.r)];
            f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m);
            l += f * ml.y;
            lr += f * ml.z;
        }
        const int n = min(PARTS, part.y + 1 - c0);
#pragma unroll 2
        for (int k = 0; k < n; ++k) {
            const float4 *src = (const float4 *)(a.ws_o + part_row(c0 + k, part.x, rows_tile, r0) * D);
#pragma unroll
            for (int rr = 0; rr < R; ++rr) {
                const float fk = __shfl_sync(0xffffffffu, f, k * R + rr);
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (rr < rows && lane + 32 * i < D / 4) merge_add(o[rr][i], src[rr * (D / 4) + lane + 32 * i], fk);
            }
        }
    }
#pragma unroll
    for (int x = R; x < 32; x <<= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, x);
        lr += __shfl_xor_sync(0xffffffffu, lr, x);
    }
    const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
#pragma unroll
    for (int rr = 0; rr < R; ++rr) {
        const float iv = __shfl_sync(0xffffffffu, inv, rr);
        const long long at = __shfl_sync(0xffffffffu, mine.at, rr);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (rr < rows && lane + 32 * i < D / 4) merge_put<D>(a, at, lane + 32 * i, o[rr][i], iv);
    }
    if (a.lse && lane < rows) a.lse[mine.at] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
}

// Lanes look at 32 parts' maxima and sums at once, so that the parts' rows are read without waiting for one another.
template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32) tree_merge_kernel(const TreeArgs a, int rows_tile) {
    const int rows_all = a.n_draft * a.group, bg = blockIdx.x / rows_all;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const MergeRow mr = merge_row(a, bg, blockIdx.x - bg * rows_all, rows_tile);
    grid_wait();
    const int2 part = a.parts[bg * a.row_tiles + mr.rt];
    if (part.x == part.y) return;
    __shared__ float4 s_o[kMergeWarps][D / 4];
    constexpr int PER = (D + 127) / 128;  // float4 of a lane
    float m = -INFINITY;
    for (int c = part.x + lane; c <= part.y; c += 32) m = fmaxf(m, a.ws_ml[part_row(c, part.x, rows_tile, mr.r)].x);
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    float l = 0.0f, lr = 0.0f;
    float4 o[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c0 = part.x; c0 <= part.y; c0 += 32) {
        float f = 0.0f;
        if (c0 + lane <= part.y) {
            const float4 ml = a.ws_ml[part_row(c0 + lane, part.x, rows_tile, mr.r)];
            f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m);
            l += f * ml.y;
            lr += f * ml.z;
        }
        const int n = min(32, part.y + 1 - c0);
#pragma unroll 4
        for (int k = warp; k < n; k += kMergeWarps) {
            const float fk = __shfl_sync(0xffffffffu, f, k);
            const float4 *src = (const float4 *)(a.ws_o + part_row(c0 + k, part.x, rows_tile, mr.r) * D);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (lane + 32 * i < D / 4) merge_add(o[i], src[lane + 32 * i], fk);
        }
    }
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, x);
        lr += __shfl_xor_sync(0xffffffffu, lr, x);
    }
    const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < D / 4) s_o[warp][lane + 32 * i] = o[i];
    __syncthreads();
    for (int i = threadIdx.x; i < D / 4; i += kMergeWarps * 32) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) merge_add(v, s_o[w][i], 1.0f);
        merge_put<D>(a, mr.at, i, v, inv);
    }
    if (a.lse && lane == 0 && warp == 0) a.lse[mr.at] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
}

// ---- host side ----
// Row tiles: a warp holds 8, 16 or (up to head_dim 128) 32 rows; more rows take four warps' 16, so that a tile
// of keys is read from memory once per 64 rows. More rows mostly go to the 5th-generation tensor cores
// (tree_tile_rows()).
enum class Shape { R8, R16, R32, R64, Tile };

Shape shape_for(const PoolView &p, int rows, bool capped) {
    const int head_dim = p.head_dim;
    if (tree_tile_rows(p, rows, capped)) return Shape::Tile;
    if (rows <= 8) return Shape::R8;
    if (rows <= 16) return Shape::R16;
    if (rows <= 32 && head_dim <= 128) return Shape::R32;
    return Shape::R64;
}
int tile_rows(Shape s, const PoolView &p, int rows, bool capped) {
    if (s == Shape::Tile) return tree_tile_rows(p, rows, capped);
    return s == Shape::R8 ? 8 : s == Shape::R16 ? 16 : s == Shape::R32 ? 32 : 64;
}

int grid_ctas(Shape s, const PoolView &p, int rows, int sms) {
    if (s == Shape::Tile) return tree_tile_ctas(p, rows, sms);
    return sms * rows_ctas(p.head_dim, p.dtype == EKV_DTYPE_Q8_0, s == Shape::R8 ? 1 : s == Shape::R32 ? 4 : 2, s == Shape::R64 ? 4 : 1);
}

struct WsLayout {
    size_t parts, ml, o, total;
};
WsLayout ws_layout(const PoolView &p, int n_batch, int rows, bool capped, int rt, int sms) {
    const Shape sh = shape_for(p, rows, capped);
    const size_t slots = 2ull * grid_ctas(sh, p, rows, sms) * tile_rows(sh, p, rows, capped);
    WsLayout w;
    w.parts = 0;
    w.ml = ((size_t)n_batch * p.kv_heads * rt * sizeof(int2) + 255) / 256 * 256;
    w.o = w.ml + slots * sizeof(float4);
    w.total = w.o + slots * p.head_dim * sizeof(float);
    return w;
}

template <int D, bool Q8, bool FINE, int NR, int WR, int WK>
int launch_rows(const TreeArgs &a, int grid, cudaStream_t s) {
    using C = Cfg<D, Q8, NR, WR, WK>;
    static std::atomic<uint64_t> smem_done{0};
    if (const int rc = allow_smem(tree_rows_kernel<D, Q8, FINE, NR, WR, WK>, C::SMEM, smem_done)) return rc;
    return launch_clusters_after(a.cluster, tree_rows_kernel<D, Q8, FINE, NR, WR, WK>, grid, C::THREADS, C::SMEM, s, a);
}

template <int D, bool Q8, bool FINE>
int launch_shape(const TreeArgs &a, Shape sh, int grid, cudaStream_t s) {
    switch (sh) {
        case Shape::R8: return launch_rows<D, Q8, FINE, 1, 1, 4>(a, grid, s);
        case Shape::R16: return launch_rows<D, Q8, FINE, 2, 1, 4>(a, grid, s);
        case Shape::R32:
            if constexpr (D <= 128) return launch_rows<D, Q8, FINE, 4, 1, 4>(a, grid, s);
            return EKV_ERR_UNSUPPORTED;
        default:  // (bf16 at head_dim 128: 33 rows and more are the tile kernel's)
            if constexpr (Q8 || D != 128) return launch_rows<D, Q8, FINE, 2, 4, 1>(a, grid, s);
            return EKV_ERR_UNSUPPORTED;
    }
}

template <int D>
int launch_dim(const TreeArgs &a, Shape sh, int grid, cudaStream_t s) {
    int rc;
    if (sh == Shape::Tile) {
        rc = launch_tree_tile(a, grid, s);
    } else if (a.pool.dtype == EKV_DTYPE_Q8_0) {
        if constexpr (D % 32 == 0) rc = launch_shape<D, true, true>(a, sh, grid, s);
        else rc = EKV_ERR_UNSUPPORTED;
    } else {
        rc = a.out_dtype == EKV_DTYPE_F32 ? launch_shape<D, false, true>(a, sh, grid, s) : launch_shape<D, false, false>(a, sh, grid, s);
    }
    if (rc || !a.split) return rc;
    const int tr = tile_rows(sh, a.pool, a.n_draft * a.group, a.cap_log2 != 0.0f);
    const int rows = a.n_draft * a.group, n_rows = a.n_batch * a.pool.kv_heads * rows;
    // A warp for four rows once that leaves two warps to each place of a CTA; rows are then many and their parts few (16384
    // rows of two or three parts 82.8 us for the call, with a block for each 123; 4096 rows 59.4 and 63.6; 780 rows of
    // sixteen parts 34 and 20; 512 rows 153 and 151).
    if (n_rows >= 2 * kMergeWarps * grid) {
        const int n_groups = a.n_batch * a.pool.kv_heads * ((rows + kMergeRows - 1) / kMergeRows);
        return launch_after(tree_merge_rows_kernel<D>, (n_groups + kMergeWarps - 1) / kMergeWarps, kMergeWarps * 32, 0, s, a, tr, n_groups);
    }
    return launch_after(tree_merge_kernel<D>, n_rows, kMergeWarps * 32, 0, s, a, tr);
}

}  // namespace

size_t tree_workspace(const PoolView &p, int n_batch, int n_draft, int q_heads, bool capped, int sms) {
    const int rows = n_draft * (q_heads / p.kv_heads);
    const int tr = tile_rows(shape_for(p, rows, capped), p, rows, capped);
    return ws_layout(p, n_batch, rows, capped, (rows + tr - 1) / tr, sms).total;
}

int launch_tree_attention(TreeArgs a, int max_len, void *ws, size_t ws_bytes, int sms, cudaStream_t s) {
    const int rows = a.n_draft * a.group;
    const bool capped = a.cap_log2 != 0.0f;
    const Shape sh = shape_for(a.pool, rows, capped);
    const int tr = tile_rows(sh, a.pool, rows, capped);
    a.row_tiles = (rows + tr - 1) / tr;
    const int64_t units = (int64_t)a.n_batch * a.pool.kv_heads * a.row_tiles;
    const int64_t all_rows = (int64_t)a.n_batch * a.pool.kv_heads * rows;
    const WsLayout w = ws_layout(a.pool, a.n_batch, rows, capped, a.row_tiles, sms);
    // (a request's tiles: 64 keys, and 64 or 32 drafts; the sums of a split call are 32-bit)
    const int64_t unit_tiles = (max_len + kTile - 1) / kTile + 1;
    const int64_t most_tiles = ((int64_t)a.pool.max_blocks_per_seq * a.pool.block_tokens + kTile - 1) / kTile + 2;
    if (units > INT32_MAX || all_rows > INT32_MAX) return EKV_ERR_INVALID_ARG;
    const int full = grid_ctas(sh, a.pool, rows, sms);
    // Three ways to share the work: a CTA per unit (one or two tiles, or many units without a workspace); a cluster of
    // CTAs per unit; CTAs with equal ranges of all tiles and a second kernel that joins the parts. The last is the most
    // even one, but its second launch costs about 3.4 us, the time of `worth` tiles: one token over 816 keys takes 9.3 us
    // with it and 8.4 as a cluster of eight, 64 requests of an 8-bit cache 22 and 20. max_len stands for the call's lengths,
    // which are on the device: where an idle sequence of 60000 tokens makes it too long the split is taken for the clusters'
    // calls as well (that token 9.9 us, the 64 requests 23.5, in bf16 18.8 for 13.5); the caller's max_prefix puts it right.
    const bool can_split = ws != nullptr && ws_bytes >= w.total && units * most_tiles < INT32_MAX;
    const int64_t even = (units * unit_tiles + full - 1) / full;  // tiles per CTA when split
    const int64_t worth = a.pool.dtype == EKV_DTYPE_Q8_0 ? 1 : 3;
    a.split = 0;
    a.cluster = 1;
    if (unit_tiles > 2) {
        int c = 1;
        const bool few = sh != Shape::Tile && tr * a.pool.head_dim <= 2048;  // what Cfg::CLUSTERS has room for
        if (few)
            while (c < kMaxCluster && 2 * c <= unit_tiles && units * 2 * c <= full) c *= 2;
        if (c > 1 && (!can_split || (unit_tiles + c - 1) / c <= even + worth)) a.cluster = c;
        else a.split = can_split;
    }
    int64_t grid = units * a.cluster;
    if (a.split) {
        grid = std::min<int64_t>(full, units * unit_tiles);
        a.parts = (int2 *)ws;
        a.ws_ml = (float4 *)((uint8_t *)ws + w.ml);
        a.ws_o = (float *)((uint8_t *)ws + w.o);
    }
    if (grid > INT32_MAX) return EKV_ERR_INVALID_ARG;
    switch (a.pool.head_dim) {
        case 48: return launch_dim<48>(a, sh, (int)grid, s);
        case 64: return launch_dim<64>(a, sh, (int)grid, s);
        case 128: return launch_dim<128>(a, sh, (int)grid, s);
        case 256: return launch_dim<256>(a, sh, (int)grid, s);
        default: return EKV_ERR_UNSUPPORTED;
    }
}

}  // namespace ekv
