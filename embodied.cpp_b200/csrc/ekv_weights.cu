// ekv_weights.cu -- the attention weight that each cached key got from a call's query rows:
//   w[b][h][k] = decay * w[b][h][k] + sum over rows r of KV head h of exp(s_rk - lse_r)
// with the scores s and the lse of ekv_tree_attention. Every key's sum is one CTA's, in a fixed order: no
// atomics, the same result every time. K is read once, V not at all.
#include <algorithm>
#include <type_traits>

#include "ekv_decode.cuh"

namespace ekv {
namespace {

using namespace decode;
using namespace sm100;

constexpr int kWarps = 4;  // 16 keys of a 64-key tile each
constexpr int kThreads = kWarps * 32 + 32;
constexpr int kMaxStages = 8;

template <int D, bool Q8>
struct WCfg {
    using T = TileCfg<D, Q8>;
    static constexpr int STAGE = (T::KV_BYTES + 1023) / 1024 * 1024;
    static constexpr int QROW = q_row_bytes<D>();
    static constexpr int QROWS = D > 128 ? 128 : 256;        // query rows held at a time
    // two CTAs per SM: what their query rows leave of half an SM's shared memory holds tiles in flight
    static constexpr int fixed(int rows) { return rows * (QROW + 4) + 1024 + 1024; }
    static constexpr int stages(int rows) {
        const int n = (112 * 1024 - fixed(rows)) / STAGE;
        return n < 2 ? 2 : n > kMaxStages ? kMaxStages : n;
    }
    static constexpr int smem(int rows) { return stages(rows) * STAGE + fixed(rows); }
};

struct WShared {
    uint64_t full[kMaxStages], empty[kMaxStages];
    RangeScratch range;
    int abort;
    int table[kTableWindow];
};

template <int D, bool Q8>
__global__ void __launch_bounds__(kThreads, 2) key_weights_kernel(const TreeArgs a, int q_rows, int nst) {
    using C = WCfg<D, Q8>;
    using T = TileCfg<D, Q8>;
    constexpr int KS = D / 16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    static_assert(sizeof(WShared) <= 1024, "barrier block");
    WShared &sh = *(WShared *)(smem + nst * C::STAGE);
    uint8_t *sq = smem + nst * C::STAGE + 1024;           // [q_rows] rows of C::QROW bytes
    float *slse = (float *)(sq + q_rows * C::QROW);       // [q_rows] lse in the log2 domain
    volatile int *abort = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hk = a.pool.kv_heads, rows_all = a.n_draft * a.group;

    if (threadIdx.x == 0) {
        for (int i = 0; i < nst; ++i) {
            mbar_init(smem_addr(&sh.full[i]), 1);
            mbar_init(smem_addr(&sh.empty[i]), kWarps);
        }
        sh.abort = 0;
        mbar_init_fence();
    }
    auto request = [&](int b, bool report) {
        Req r = load_req(a, b, report);
        if (r.n_prefix > a.weight_stride) {  // no room for its weights
            if (report) report_error(a.pool.status, DEV_ERR_BAD_POS, b, r.n_prefix, 6);
            r.n_prefix = (int)a.weight_stride;
        }
        return r;
    };
    grid_wait();
    const Range rg = find_range<kThreads>(a.n_batch, hk, sh.range, [&](int b) {
        return (request(b, false).n_prefix + kTile - 1) / kTile;
    });

    int st = 0, turn = 0;  // stage of the next tile, and how often the ring went round
    auto advance = [&]() {
        if (++st == nst) {
            st = 0;
            ++turn;
        }
    };
    bool ok = true;
    TableWindow tw;  // (the feeder's)
    tw.reset(sh.table);
    int b = rg.b;
    uint32_t base = rg.base;
    Req rq{};
    int rq_of = -1;  // the request that rq describes
    for (uint32_t x = rg.lo; x < rg.hi && b < a.n_batch;) {
        if (b != rq_of) rq = request(b, warp == 0), rq_of = b;
        const int n_tiles = (rq.n_prefix + kTile - 1) / kTile;
        const uint32_t span = (uint32_t)n_tiles * hk;
        if (x >= base + span) {
            base += span;
            ++b;
            continue;
        }
        const int g = (int)((x - base) / (uint32_t)n_tiles);
        const int t0 = (int)(x - base) - g * n_tiles;
        const int t1 = min(n_tiles, t0 + (int)(rg.hi - x));

        for (int c0 = 0; c0 < rows_all; c0 += q_rows) {
            const int rows = min(q_rows, (rows_all - c0 + 15) / 16 * 16);
            if (warp == kWarps) {
                // ---- feeder ----
                Piece next = find_piece<D, Q8>(a, rq, g, t0 * kTile, tw, lane);
                for (int j = t0; j < t1; ++j, advance()) {
                    const Piece pc = next;
                    if (j + 1 < t1) next = find_piece<D, Q8>(a, rq, g, (j + 1) * kTile, tw, lane);
                    if (turn > 0) ok = ok && warp_wait(smem_addr(&sh.empty[st]), (turn - 1) & 1, abort);
                    if (!ok) {
                        *abort = 1;
                        continue;
                    }
                    issue_piece<D, Q8, false>(a, pc, smem_addr(smem + st * C::STAGE), 0, smem_addr(&sh.full[st]), 0, lane);
                }
                continue;
            }
            // ---- query rows c0 .. c0 + rows to shared memory, in the products' column order ----
            asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");  // the last rows are done with
            {
                // a warp takes 32 / U rows at a time, a lane one 16-byte unit (or two) of them
                constexpr int U = D / 8, UL = U < 32 ? U : 32, PER = 32 / UL;
                const int sub = lane / UL;
#pragma unroll 4
                for (int r = warp * PER + sub; r < rows; r += kWarps * PER) {
                    const int row = c0 + r, t = row / a.group;
                    const bool on = sub < PER && row < rows_all && t < rq.n_nodes;
                    const uint4 *src = (const uint4 *)(a.q + (((long long)b * a.n_draft + t) * a.q_heads + g * a.group + row - t * a.group) * D);
#pragma unroll
                    for (int u = lane % UL; u < U; u += UL) {
                        const uint4 v = on ? __ldg(src + u) : make_uint4(0, 0, 0, 0);
                        if (sub < PER) store_q_unit<Q8>(sq + r * C::QROW, u, v);
                    }
                }
            }
            for (int r = threadIdx.x; r < rows; r += kWarps * 32) {
                const int row = c0 + r, t = row / a.group;
                float l = INFINITY;  // no such row, or one that saw nothing: weight 0
                if (row < rows_all && t < rq.n_nodes) {
                    l = a.lse[((long long)b * a.n_draft + t) * a.q_heads + g * a.group + row - t * a.group] * 1.4426950408889634f;
                    if (l == -INFINITY) l = INFINITY;
                }
                slse[r] = l;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");

            const int rq0 = lane >> 2, c = lane & 3;
            const ScoreFn score{a.scale_log2, a.cap_log2, a.cap_in};
            const int key_l = 16 * warp + 8 * ((rq0 >> 1) & 1) + 2 * c + (rq0 & 1);  // the key this lane writes (rq0 < 4)
            float *wrow = a.weights + ((long long)b * hk + g) * a.weight_stride;
            // the entry this lane adds to, a tile ahead
            auto load_old = [&](int j) {
                const int key = j * kTile + key_l;
                return rq0 < 4 && key < rq.n_prefix && j < t1 && (c0 > 0 || a.decay != 0.0f) ? wrow[key] : 0.0f;
            };
            float next_old = load_old(t0);
            for (int j = t0; j < t1; ++j, advance()) {
                const int par = turn & 1;
                const uint32_t sk = smem_addr(smem + st * C::STAGE);
                const int key = j * kTile + key_l;
                const bool writes = rq0 < 4 && key < rq.n_prefix;
                const float old = next_old;
                next_old = load_old(j + 1);
                ok = ok && warp_wait(smem_addr(&sh.full[st]), par, abort);
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                const int key0 = 16 * warp;
                uint32_t kf[KS][4];
                float sc[Q8 ? KS / 2 : 1][2][2];  // scales of the lane's keys by group
                if constexpr (!Q8) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) load_k_step<D>(sk, key0, ks, lane, kf[ks]);
                } else {
#pragma unroll
                    for (int gr = 0; gr < KS / 2; ++gr)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const uint2 w = lds64(sk + q8_qs_off(key0 + 8 * n + rq0, 32 * gr + 8 * c, D));
                            int8x4_to_bf16(w.x, kf[2 * gr][2 * n], kf[2 * gr][2 * n + 1]);
                            int8x4_to_bf16(w.y, kf[2 * gr + 1][2 * n], kf[2 * gr + 1][2 * n + 1]);
                            const int krow = key0 + 8 * n + 2 * c;
                            sc[gr][n][0] = lds_f16(sk + T::SCALES + (krow * T::G32 + gr) * 2);
                            sc[gr][n][1] = lds_f16(sk + T::SCALES + ((krow + 1) * T::G32 + gr) * 2);
                        }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&sh.empty[st]));  // the keys are in registers
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // keys (n, e): 8 n + 2 c + e, rows of this lane
                // two 16-row tiles at a time: their products do not wait for one another
                auto row_tiles = [&](auto count, int r0) {
                    constexpr int M = decltype(count)::value;
                    float s[M][2][4];
#pragma unroll
                    for (int m = 0; m < M; ++m)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[m][n][i] = 0.0f;
                    const uint32_t qa = smem_addr(sq) + (r0 + (lane & 15)) * C::QROW + (lane >> 4) * 16;
                    if constexpr (!Q8) {
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                            for (int m = 0; m < M; ++m) {
                                uint32_t qf[4];
                                ldmatrix_x4(qf, qa + m * 16 * C::QROW + 32 * ks);
                                mma_bf16(s[m][0], qf, kf[ks][0], kf[ks][1]);
                                mma_bf16(s[m][1], qf, kf[ks][2], kf[ks][3]);
                            }
                    } else {
#pragma unroll
                        for (int gr = 0; gr < KS / 2; ++gr)
#pragma unroll
                            for (int m = 0; m < M; ++m) {
                                uint32_t q0[4], q1[4];
                                ldmatrix_x4(q0, qa + m * 16 * C::QROW + 64 * gr);
                                ldmatrix_x4(q1, qa + m * 16 * C::QROW + 64 * gr + 32);
#pragma unroll
                                for (int n = 0; n < 2; ++n) {
                                    float p[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                    mma_bf16(p, q0, kf[2 * gr][2 * n], kf[2 * gr][2 * n + 1]);
                                    mma_bf16(p, q1, kf[2 * gr + 1][2 * n], kf[2 * gr + 1][2 * n + 1]);
                                    s[m][n][0] = fmaf(p[0], sc[gr][n][0], s[m][n][0]);
                                    s[m][n][1] = fmaf(p[1], sc[gr][n][1], s[m][n][1]);
                                    s[m][n][2] = fmaf(p[2], sc[gr][n][0], s[m][n][2]);
                                    s[m][n][3] = fmaf(p[3], sc[gr][n][1], s[m][n][3]);
                                }
                            }
                    }
#pragma unroll
                    for (int m = 0; m < M; ++m) {
                        const float l0 = slse[r0 + 16 * m + rq0], l1 = slse[r0 + 16 * m + rq0 + 8];
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                acc[2 * n + e] += ex2(score(s[m][n][e]) - l0) + ex2(score(s[m][n][2 + e]) - l1);
                    }
                };
                int r0 = 0;
#pragma unroll 1
                for (; r0 + 32 <= rows; r0 += 32) row_tiles(std::integral_constant<int, 2>(), r0);
                if (r0 < rows) row_tiles(std::integral_constant<int, 1>(), r0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int m = 4; m < 32; m <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], m);
                const float mine = rq0 & 2 ? (rq0 & 1 ? acc[3] : acc[2]) : (rq0 & 1 ? acc[1] : acc[0]);
                if (writes) wrow[key] = old * (c0 > 0 ? 1.0f : a.decay) + mine;
            }
        }
        x += t1 - t0;
    }
    if (!ok && lane == 0) report_error(a.pool.status, DEV_ERR_TIMEOUT, blockIdx.x, warp, 8);
    if (warp == kWarps && !ok && lane == 0) {
        for (int st = 0; st < nst; ++st) {  // leave no copy writing this CTA's shared memory
            mbar_wait_drain(smem_addr(&sh.full[st]), 0, kWait / 64);
            mbar_wait_drain(smem_addr(&sh.full[st]), 1, kWait / 64);
        }
    }
}

template <int D, bool Q8>
int launch(const TreeArgs &a, int max_len, int sms, cudaStream_t s) {
    using C = WCfg<D, Q8>;
    const int64_t rows = (int64_t)a.n_draft * a.group;
    const int q_rows = (int)std::min<int64_t>((rows + 15) / 16 * 16, C::QROWS);
    const int smem = C::smem(q_rows);
    static std::atomic<uint64_t> smem_done{0};
    if (const int rc = allow_smem(key_weights_kernel<D, Q8>, 227 * 1024, smem_done)) return rc;
    const int64_t most = ((int64_t)a.pool.max_blocks_per_seq * a.pool.block_tokens + kTile - 1) / kTile;
    if ((int64_t)a.n_batch * a.pool.kv_heads * most > INT32_MAX) return EKV_ERR_UNSUPPORTED;
    const int64_t tiles = (int64_t)a.n_batch * a.pool.kv_heads * ((max_len + kTile - 1) / kTile);
    const int ctas = smem > 112 * 1024 ? 1 : 2;
    const int grid = (int)std::min<int64_t>((int64_t)sms * ctas, std::max<int64_t>(1, tiles));
    return launch_after(key_weights_kernel<D, Q8>, grid, kThreads, smem, s, a, q_rows, C::stages(q_rows));
}

template <int D>
int launch_dim(const TreeArgs &a, int max_len, int sms, cudaStream_t s) {
    if (a.pool.dtype != EKV_DTYPE_Q8_0) return launch<D, false>(a, max_len, sms, s);
    if constexpr (D % 32 == 0) return launch<D, true>(a, max_len, sms, s);
    return EKV_ERR_UNSUPPORTED;
}

}  // namespace

int launch_key_weights(const TreeArgs &a, int max_len, int sms, cudaStream_t s) {
    switch (a.pool.head_dim) {
        case 48: return launch_dim<48>(a, max_len, sms, s);
        case 64: return launch_dim<64>(a, max_len, sms, s);
        case 128: return launch_dim<128>(a, max_len, sms, s);
        case 256: return launch_dim<256>(a, max_len, sms, s);
        default: return EKV_ERR_UNSUPPORTED;
    }
}

}  // namespace ekv
