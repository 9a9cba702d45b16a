// ekv_weights.cu -- the attention weight that each cached key got from a call's query rows:
//   w[b][h][k] = decay * w[b][h][k] + sum over rows r of KV head h of exp(s_rk - lse_r)
// with the scores s and the lse of ekv_tree_attention. Every key's sum is one CTA's, in a fixed order: no
// atomics, the same result every time. K is read once, V not at all.
// Keys are the rows of the products (S^T = K Q^T), so that a lane holds two keys and sums over query rows in its own
// registers; with query rows as rows, twelve shuffles per tile made the consumer the bound (97 us for 16 x 16k keys).
// Bound and figures: the bytes of K up to about 16 rows of a KV head: 16 requests of 16 k keys, 8 KV heads of 128 columns
// in bf16 (503 MB), 4 rows each, take 85 us on the device, 5.9 TB/s, 90% of the measured copy rate. With more rows the matrix
// instructions and one exponential per row and key: 256 rows over 8 requests of 4096 such keys 77 us (a tcgen05 form
// would have 15 of exponentials and 11 of products). 132 rows over 4 requests of 4 k Q8_0 keys: 15.2 us.
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
constexpr int kRowTiles = 2;  // tiles of eight query rows whose products run side by side

template <int D, bool Q8>
struct WCfg {
    using T = TileCfg<D, Q8>;
    static constexpr int STAGE = (T::KV_BYTES + 1023) / 1024 * 1024;
    static constexpr int QROW = q_row_bytes<D, Q8>();
    static constexpr int QROWS = D > 128 ? 128 : 256;        // query rows held at a time
    // CTAs per SM by their registers (the keys' 16 rows are D / 4 of them); what their query rows leave of the shared
    // memory holds tiles in flight
    static constexpr int CTAS = D > 128 ? 2 : 3, ROOM = (CTAS == 2 ? 112 : 74) * 1024;
    static constexpr int fixed(int rows) { return rows * (QROW + 4) + 1024 + 1024; }
    static constexpr int stages(int rows) {
        const int n = (ROOM - fixed(rows)) / STAGE;
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
__global__ void __launch_bounds__(kThreads, WCfg<D, Q8>::CTAS) key_weights_kernel(const TreeArgs a, int q_rows, int nst) {
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
    const Range rg = find_range<kThreads>(
        a.n_batch, hk, sh.range, [&](int b) { return request(b, blockIdx.x == 0); },
        [](const Req &r) { return (r.n_prefix + kTile - 1) / kTile; });

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
    Req rq = rg.req;
    int rq_of = b;  // the request that rq describes
    for (uint32_t x = rg.lo; x < rg.hi && b < a.n_batch;) {
        if (b != rq_of) rq = request(b, true), rq_of = b;
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
            const int rows = min(q_rows, (rows_all - c0 + 7) / 8 * 8);
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
                    // the weights that this tile adds to: from memory to L2 while the tile is on its way (3 lines of 128
                    // bytes hold 64 of them at any alignment)
                    if (lane < 3 && (c0 > 0 || a.decay != 0.0f)) {
                        const float *w = a.weights + ((long long)b * hk + g) * a.weight_stride + j * kTile + lane * 32;
                        if (j * kTile + lane * 32 < rq.n_prefix) asm volatile("prefetch.global.L2 [%0];" ::"l"(w));
                    }
                    issue_piece<D, Q8, false>(a, pc, smem_addr(smem + st * C::STAGE), 0, smem_addr(&sh.full[st]), 0, lane);
                }
                continue;
            }
            // ---- query rows c0 .. c0 + rows to shared memory, in the products' column order ----
            asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");  // the last rows are done with
            stage_q_rows<D, Q8>(smem_addr(sq), rows, a.q, warp, kWarps, lane, [&](int r) -> const uint16_t * {
                const int row = c0 + r, t = row_token(a, row);
                if (row >= rows_all || t >= rq.n_nodes) return nullptr;
                return a.q + (((long long)b * a.n_draft + t) * a.q_heads + g * a.group + row - t * a.group) * D;
            });
            for (int r = threadIdx.x; r < rows; r += kWarps * 32) {
                const int row = c0 + r, t = row_token(a, row);
                float l = INFINITY;  // no such row, or one that saw nothing: weight 0
                if (row < rows_all && t < rq.n_nodes) {
                    l = a.lse[((long long)b * a.n_draft + t) * a.q_heads + g * a.group + row - t * a.group] * 1.4426950408889634f;
                    if (l == -INFINITY) l = INFINITY;
                }
                slse[r] = l;
            }
            cp_async_wait_all();
            asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");

            const int kq = lane >> 2, c = lane & 3;  // keys kq and kq + 8, query rows 2 c and 2 c + 1 of a lane's elements
            const ScoreFn score{a.scale_log2, a.cap_log2, a.cap_in};
            const int key_l = 16 * warp + kq + 8 * (c & 1);  // the key this lane writes (c < 2)
            float *wrow = a.weights + ((long long)b * hk + g) * a.weight_stride;
            // the entry this lane adds to, a tile ahead
            auto load_old = [&](int j) {
                const int key = j * kTile + key_l;
                return c < 2 && key < rq.n_prefix && j < t1 && (c0 > 0 || a.decay != 0.0f) ? wrow[key] : 0.0f;
            };
            float next_old = load_old(t0);
            for (int j = t0; j < t1; ++j, advance()) {
                const int par = turn & 1;
                const uint32_t sk = smem_addr(smem + st * C::STAGE);
                const int key = j * kTile + key_l;
                const bool writes = c < 2 && key < rq.n_prefix;
                const float old = next_old;
                next_old = load_old(j + 1);
                ok = ok && warp_wait(smem_addr(&sh.full[st]), par, abort);
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                const int key0 = 16 * warp;
                uint32_t kf[KS][4];
                uint32_t sc0[Q8 ? (T::G32 + 1) / 2 : 1], sc1[Q8 ? (T::G32 + 1) / 2 : 1];  // scales of keys kq, kq + 8
                if constexpr (!Q8) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) load_k_rows<D>(sk, key0, ks, lane, kf[ks]);
                } else {
#pragma unroll
                    for (int gr = 0; gr < KS / 2; ++gr) {
                        const uint2 w0 = lds64(sk + q8_qs_off(key0 + kq, 32 * gr + 8 * c, D));
                        const uint2 w1 = lds64(sk + q8_qs_off(key0 + kq + 8, 32 * gr + 8 * c, D));
                        int8x4_to_bf16(w0.x, kf[2 * gr][0], kf[2 * gr][2]);
                        int8x4_to_bf16(w1.x, kf[2 * gr][1], kf[2 * gr][3]);
                        int8x4_to_bf16(w0.y, kf[2 * gr + 1][0], kf[2 * gr + 1][2]);
                        int8x4_to_bf16(w1.y, kf[2 * gr + 1][1], kf[2 * gr + 1][3]);
                    }
                    load_scales<T::G32>(sk + T::SCALES + (key0 + kq) * T::G32 * 2, sc0);
                    load_scales<T::G32>(sk + T::SCALES + (key0 + kq + 8) * T::G32 * 2, sc1);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&sh.empty[st]));  // the keys are in registers
                float acc0, acc1;
                // M tiles of eight query rows at a time: their products do not wait for one another
                auto row_tiles = [&](auto count, auto checked, int r0) {
                    constexpr int M = decltype(count)::value;
                    float s[M][2][4];  // even and odd column steps (Q8_0: one sum of scaled groups)
#pragma unroll
                    for (int m = 0; m < M; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[m][0][i] = s[m][1][i] = 0.0f;
                    const uint32_t qa = smem_addr(sq) + r0 * C::QROW;
#pragma unroll
                    for (int i = 0; i < (KS + 1) / 2; ++i) {
                        uint32_t f[M][4];
#pragma unroll
                        for (int m = 0; m < M; ++m) load_q_steps<D, Q8>(qa + m * 8 * C::QROW, i, lane, f[m]);
                        if constexpr (!Q8) {
#pragma unroll
                            for (int m = 0; m < M; ++m) mma_bf16(s[m][0], kf[2 * i], f[m][0], f[m][1]);
                            if (2 * i + 1 < KS) {
#pragma unroll
                                for (int m = 0; m < M; ++m) mma_bf16(s[m][1], kf[2 * i + 1], f[m][2], f[m][3]);
                            }
                        } else {
                            float p[M][4];
#pragma unroll
                            for (int m = 0; m < M; ++m) {
                                p[m][0] = p[m][1] = p[m][2] = p[m][3] = 0.0f;
                                mma_bf16(p[m], kf[2 * i], f[m][0], f[m][1]);
                            }
#pragma unroll
                            for (int m = 0; m < M; ++m) mma_bf16(p[m], kf[2 * i + 1], f[m][2], f[m][3]);
                            const float f0 = scale_of(sc0, i), f1 = scale_of(sc1, i);
#pragma unroll
                            for (int m = 0; m < M; ++m) {
                                s[m][0][0] = fmaf(p[m][0], f0, s[m][0][0]);
                                s[m][0][1] = fmaf(p[m][1], f0, s[m][0][1]);
                                s[m][0][2] = fmaf(p[m][2], f1, s[m][0][2]);
                                s[m][0][3] = fmaf(p[m][3], f1, s[m][0][3]);
                            }
                        }
                    }
                    float x[M][4];
#pragma unroll
                    for (int m = 0; m < M; ++m)
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[m][k] = s[m][0][k] + s[m][1][k];
                    score(*(float(*)[4 * M])x);
#pragma unroll
                    for (int m = 0; m < M; ++m) {
                        const float2 l = *(const float2 *)&slse[r0 + 8 * m + 2 * c];
                        if constexpr (decltype(checked)::value) {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if ((k & 1 ? l.y : l.x) == INFINITY) x[m][k] = -INFINITY;
                        }
                        acc0 += ex2(x[m][0] - l.x) + ex2(x[m][1] - l.y);
                        acc1 += ex2(x[m][2] - l.x) + ex2(x[m][3] - l.y);
                    }
                };
                // the sum of key key_l over all rows (checked: tile by tile, in the same order)
                auto sum_rows = [&](auto checked) {
                    acc0 = acc1 = 0.0f;
                    int r0 = 0;
                    if constexpr (!decltype(checked)::value)
#pragma unroll 1
                        for (; r0 + 8 * kRowTiles <= rows; r0 += 8 * kRowTiles) row_tiles(std::integral_constant<int, kRowTiles>(), checked, r0);
#pragma unroll 1
                    for (; r0 < rows; r0 += 8) row_tiles(std::integral_constant<int, 1>(), checked, r0);
#pragma unroll
                    for (int m = 1; m < 4; m <<= 1) {
                        acc0 += __shfl_xor_sync(0xffffffffu, acc0, m);
                        acc1 += __shfl_xor_sync(0xffffffffu, acc1, m);
                    }
                    return c & 1 ? acc1 : acc0;
                };
                // Rows that do not count have lse inf, and a number less inf is nothing. A key that is not finite has no
                // number with them: a sum that came out NaN is taken again without them. (With that select in every sum
                // 16 x 16 k keys took 86.8 us instead of 84.8, 256 rows 79.8 instead of 76.8.)
                float mine = sum_rows(std::false_type());
                if (__any_sync(0xffffffffu, writes && mine != mine)) mine = sum_rows(std::true_type());
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
    const int q_rows = (int)std::min<int64_t>((rows + 7) / 8 * 8, C::QROWS);
    const int smem = C::smem(q_rows);
    static std::atomic<uint64_t> smem_done{0};
    if (const int rc = allow_smem(key_weights_kernel<D, Q8>, 227 * 1024, smem_done)) return rc;
    const int64_t most = ((int64_t)a.pool.max_blocks_per_seq * a.pool.block_tokens + kTile - 1) / kTile;
    if ((int64_t)a.n_batch * a.pool.kv_heads * most > INT32_MAX) return EKV_ERR_UNSUPPORTED;
    const int64_t tiles = (int64_t)a.n_batch * a.pool.kv_heads * ((max_len + kTile - 1) / kTile);
    const int ctas = std::min(C::CTAS, 227 * 1024 / (smem + 1024));
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
