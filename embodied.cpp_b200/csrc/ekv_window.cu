// ekv_window.cu -- attention of appended rows over the pool with a sliding window and first tokens that stay visible.
//
// A row at slot p sees the slots k <= p with k > p - window or k < sinks: out = sum_k p_k v_k / sum_k p_k, p_k = exp(scale q.k - m).
// This file has the kernel for few rows of a KV head (single tokens, mostly), the choice between it and the tile kernel, and the
// join of units that several CTAs took parts of.
//
// window_rows_kernel: as tree_rows_kernel (ekv_tree.cu says more), over the keys that the unit's rows see and no others. Products are
// transposed, S^T = K Q^T and O^T = V^T P^T on mma.sync, so that 16 keys (or value columns) and 8 rows fill an instruction; four
// warps take 16 keys of a 64-key tile each and keep their rows' maxima, sums and outputs in registers; one warp feeds tiles through
// the copy engine. P is rounded to bf16 and the row divided by the sum of the rounded ones; over 8-bit pages p times the value's scale
// is two bf16 parts, so that a heavy key's 32 columns are not all off by the same 2^-8.
#include <algorithm>
#include <type_traits>

#include "ekv_window.cuh"

namespace ekv {
namespace {

using namespace decode;
using namespace sm100;
using namespace window;

constexpr int kMaxCluster = 8, kKeyWarps = 4, kFewRows = 16;

constexpr int few_ctas(int d, bool q8, int nr) { return d * nr > 256 || (d > 128 && !q8) ? 1 : 2; }

// 8 * NR rows; kKeyWarps warps of 16 keys, and one feeder warp.
template <int D, bool Q8, int NR>
struct FCfg {
    using T = TileCfg<D, Q8>;
    static constexpr int NC = kKeyWarps * 32, THREADS = NC + 32, ROWS = 8 * NR;
    static constexpr int STAGE = (2 * T::KV_BYTES + 1023) / 1024 * 1024, V_OFF = T::KV_BYTES;
    static constexpr int X_COLS = (NR == 1 ? 128 : 64) < D ? (NR == 1 ? 128 : 64) : D;  // columns joined at a time: 16 KB of rows
    static constexpr int X_BYTES = kKeyWarps * ROWS * X_COLS * 4, ML_BYTES = kKeyWarps * ROWS * 16;
    static constexpr bool Q_SMEM = D * NR > 256;
    static constexpr int Q_BYTES = Q_SMEM ? ROWS * q_row_bytes<D, Q8>() : 0;
    static constexpr bool CLUSTERS = ROWS * D <= 2048;
    static constexpr int P_BYTES = CLUSTERS ? ROWS * D * 4 + kMaxCluster * (ROWS + 1) * 16 : 0;
    static constexpr int FIXED = X_BYTES + ML_BYTES + Q_BYTES + P_BYTES + 1024 + 1024;
    static constexpr int CTAS = few_ctas(D, Q8, NR), BUDGET = CTAS == 2 ? 112 * 1024 : 220 * 1024;
    static constexpr int NST_FIT = (BUDGET - FIXED) / STAGE, NST = NST_FIT > 8 ? 8 : NST_FIT;
    static constexpr int SMEM = NST * STAGE + FIXED;
    static_assert(NST >= 2, "two stages");
};

// Block ids of the entries that a request's rows see, in the order of their keys: the first `front` entries of its table, then those from
// the window's on, as one list, of which kTableWindow are in shared memory. (Two lists, read 32 entries at a time, took 2.3 us before the
// first tile of a row with a window of 1024 and blocks of 16 was on its way; one, with all loads at once, 1.) Used by one warp.
struct SeenBlocks {
    int *blocks;
    int request, front, skip, lo, n;
    __device__ __forceinline__ void reset(int *mem) {
        blocks = mem;
        request = -1;
    }
    __device__ __forceinline__ int place(int entry) const { return entry < front ? entry : entry - skip; }
    // Entries [first, last] of the request, of which all up to `end` will be wanted in turn.
    __device__ __forceinline__ void want(const PoolView &p, int b, int seq, const Span &sp, int first, int last, int end, int lane) {
        if (b != request) {
            auto entry = [&](int slot) { return p.bt_shift >= 0 ? slot >> p.bt_shift : slot / p.block_tokens; };
            request = b;
            front = sp.front > 0 ? entry(sp.front - 1) + 1 : 0;
            skip = max(0, entry(sp.lo) - front);
            n = 0;
        }
        first = place(first);
        if (n > 0 && first >= lo && place(last) < lo + n) return;
        __syncwarp();
        lo = first;
        n = min(kTableWindow, place(end) + 1 - first);
        int e[kTableWindow / 32], v[kTableWindow / 32];
#pragma unroll
        for (int j = 0; j < kTableWindow / 32; ++j) {
            const int i = first + lane + 32 * j;
            e[j] = i < front ? i : i + skip;
            v[j] = lane + 32 * j < n && e[j] < p.max_blocks_per_seq ? p.block_tables[(int64_t)seq * p.max_blocks_per_seq + e[j]] : -1;
        }
#pragma unroll
        for (int j = 0; j < kTableWindow / 32; ++j) {
            if (lane + 32 * j >= n) continue;
            const bool fine = v[j] >= 0 && v[j] < p.n_blocks;
            if (!fine) report_error(p.status, DEV_ERR_BAD_BLOCK, seq, e[j], v[j]);
            blocks[lane + 32 * j] = fine ? v[j] : -1;
        }
        __syncwarp();
    }
};

template <int NST>
struct FShared {
    uint64_t full_k[NST], full_v[NST], empty[NST];
    RangeScratch range;
    int abort;
    int table[kTableWindow];
};

// Column of output accumulator (16-column step ds, element i) of lane row kq (ekv_tree.cu).
template <bool Q8>
__device__ __forceinline__ int o_col(int ds, int kq, int i) {
    return Q8 ? 32 * (ds >> 1) + 4 * kq + 2 * (ds & 1) + (i >> 1) : 16 * ds + kq + 8 * (i >> 1);
}

template <int D, bool Q8, int NR>
__global__ void __launch_bounds__(FCfg<D, Q8, NR>::THREADS, FCfg<D, Q8, NR>::CTAS) window_rows_kernel(const WindowArgs a) {
    using C = FCfg<D, Q8, NR>;
    using T = TileCfg<D, Q8>;
    constexpr int NST = C::NST, KS = D / 16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float *xb = (float *)(smem + NST * C::STAGE);                  // [kKeyWarps][ROWS][X_COLS]
    float2 *sml = (float2 *)(smem + NST * C::STAGE + C::X_BYTES);  // [kKeyWarps][ROWS]: maximum, sum
    using Sh = FShared<NST>;
    static_assert(sizeof(Sh) <= 1024, "barrier block");
    Sh &sh = *(Sh *)(smem + NST * C::STAGE + C::X_BYTES + C::ML_BYTES);
    uint8_t *sq = smem + NST * C::STAGE + C::X_BYTES + C::ML_BYTES + 1024;  // [ROWS] query rows (Q_SMEM)
    float4 *part_o = (float4 *)(sq + C::Q_BYTES);              // [cluster][its share of the unit's float4 outputs]
    float4 *part_ml = part_o + C::ROWS * D / 4 + kMaxCluster;  // [cluster][ROWS]
    volatile int *abort = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = a.pool.kv_heads;

    if (threadIdx.x == 0) {
        for (int i = 0; i < NST; ++i) {
            mbar_init(smem_addr(&sh.full_k[i]), 1);
            mbar_init(smem_addr(&sh.full_v[i]), 1);
            mbar_init(smem_addr(&sh.empty[i]), kKeyWarps);
        }
        sh.abort = 0;
        mbar_init_fence();
    }
    // a unit is a request's KV head: all its rows are one row tile. Refused requests keep one (empty) tile, so that some CTA writes
    // their rows.
    auto span_of = [&](const WinReq &r) { return Span(a, r, 0, max(0, r.n - 1)); };
    auto tiles_of = [&](const WinReq &r) { return r.n == 0 ? 0 : max(1, (span_of(r).keys + kTile - 1) / kTile); };
    const int unit = blockIdx.x / a.cluster, rank = blockIdx.x - unit * a.cluster;
    if (C::CLUSTERS && a.cluster > 1) cluster_arrive_relaxed();  // (waited for before anything is sent)
    Range rg;
    grid_wait();
    grid_launch_next();
    int b = 0;
    if (a.split) {
        rg = find_range<C::THREADS>(
            a.n_batch, hk, sh.range,
            [&](int i) { return Req{0, tiles_of(load_win_req(a, i, blockIdx.x == 0)), 0}; }, [](const Req &r) { return r.n_prefix; });
        b = rg.b;
    } else {
        __syncthreads();
        b = unit / hk;
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
    SeenBlocks seen;  // (the feeder's)
    seen.reset(sh.table);
    uint32_t base = rg.base;
    WinReq rq{-1, 0, 0};
    int rq_of = -1;
    for (uint32_t x = rg.lo; (x < rg.hi || !a.split) && b < a.n_batch;) {
        if (b != rq_of) rq = load_win_req(a, b, !a.split && threadIdx.x == 0 && rank == 0 && unit == b * hk), rq_of = b;
        const int n_tiles = tiles_of(rq);
        const uint32_t span = (uint32_t)n_tiles * hk;
        if (a.split && x >= base + span) {
            base += span;
            ++b;
            continue;
        }
        const int g = a.split ? (int)((x - base) / (uint32_t)n_tiles) : unit - b * hk;
        const int t0 = a.split ? (int)(x - base) - g * n_tiles : rank * n_tiles / a.cluster;
        const int t1 = a.split ? min(n_tiles, t0 + (int)(rg.hi - x)) : (rank + 1) * n_tiles / a.cluster;
        const int rows = rq.n * a.group;
        const Span sp = span_of(rq);
        const int64_t src_row = rq.src;
        // query row r of the unit, or null where it does not take part
        auto q_row = [&](int r) -> const uint16_t * {
            const int t = row_token(a, r);
            return r < rows && rq.seq >= 0 ? a.q + (src_row + t) * a.q_stride + (int64_t)(g * a.group + r - t * a.group) * D : nullptr;
        };

        if (warp == kKeyWarps) {
            // ---- feeder: lanes 0-15 a tile's K, 16-31 its V ----
            const bool is_v = lane >= 16;
            const int last_entry = rq.seq >= 0 ? sp.last / a.pool.block_tokens : 0;
            auto find = [&](int j) {
                return find_run<kTile>(
                    a, sp, g, j * kTile, lane & 15, [&](int e0, int e1) { seen.want(a.pool, b, rq.seq, sp, e0, e1, last_entry, lane); },
                    [&](int e) { return seen.blocks[seen.place(e) - seen.lo]; });
            };
            Run next{nullptr, 0, 0, 0};
            if (t0 < t1) next = find(t0);  // (a request without rows has no tiles, and its slots mean nothing)
            if (a.split && lane == 0 && t0 == 0) {  // the CTAs of this unit: tile x is CTA ((x + 1) G - 1) / T's
                const unsigned long long end = base + (uint32_t)(g + 1) * n_tiles;
                a.parts[b * hk + g] = make_int2(blockIdx.x, (int)((end * rg.ctas - 1) / rg.total));
            }
            for (int j = t0; j < t1; ++j, advance()) {
                const Run r = next;
                if (j + 1 < t1) next = find(j + 1);
                if (turn > 0) ok = ok && warp_wait(smem_addr(&sh.empty[st]), (turn - 1) & 1, abort);
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                constexpr int ROW = Q8 ? D : 2 * D, SROW = Q8 ? D / 16 : 0;  // bytes of a row, and of its scales
                const uint32_t dst = smem_addr(smem + st * C::STAGE) + (is_v ? C::V_OFF : 0), bar = smem_addr(is_v ? &sh.full_v[st] : &sh.full_k[st]);
                const uint32_t bytes = r.src ? (uint32_t)(r.n * (ROW + SROW)) : 0u;
                const uint32_t kb = __reduce_add_sync(0xffffffffu, is_v ? 0u : bytes), vb = __reduce_add_sync(0xffffffffu, is_v ? bytes : 0u);
                if (lane == 0) {
                    mbar_arrive_expect_tx(smem_addr(&sh.full_k[st]), kb);
                    mbar_arrive_expect_tx(smem_addr(&sh.full_v[st]), vb);
                }
                __syncwarp();
                if (!r.src) continue;
                const uint8_t *src = r.src + (is_v ? (int64_t)hk * a.pool.tile_bytes : 0);
                bulk_g2s(dst + r.row * ROW, src + r.rib * ROW, (uint32_t)(r.n * ROW), bar);
                if (Q8) bulk_g2s(dst + T::SCALES + r.row * SROW, src + (int64_t)a.pool.block_tokens * D + r.rib * SROW, (uint32_t)(r.n * SROW), bar);
            }
        } else {
            // ---- rows ----
            const int wk = warp, kq = lane >> 2, c = lane & 3;  // key (or value column) and query row pair of the lane's elements
            uint32_t qf[C::Q_SMEM ? 1 : NR][C::Q_SMEM ? 1 : KS][2];
            int p_of[NR][2];  // slot of rows 8 n + 2 c (+ 1), -1 where the row does not take part
#pragma unroll
            for (int n = 0; n < NR; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 8 * n + 2 * c + e;
                    p_of[n][e] = r < rows && rq.seq >= 0 ? rq.pos0 + row_token(a, r) : -1;
                }
                if constexpr (!C::Q_SMEM) {
                    const uint16_t *src = q_row(8 * n + kq);
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int half = 0; half < 2; ++half)
                            qf[n][ks][half] = src ? __ldg((const uint32_t *)(src + q_col<Q8>(ks, c, half))) : 0u;
                }
            }
            if constexpr (C::Q_SMEM) {  // the last rows were done with at the barriers of their end
                stage_q_rows<D, Q8>(smem_addr(sq), C::ROWS, a.q, warp, kKeyWarps, lane, q_row);
                cp_async_wait_all();
                asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
            }
            auto load_q2 = [&](int n, int i, uint32_t (&f)[4]) {
                if constexpr (C::Q_SMEM) {
                    load_q_steps<D, Q8>(smem_addr(sq) + 8 * n * q_row_bytes<D, Q8>(), i, lane, f);
                } else {
                    f[0] = qf[n][2 * i][0];
                    f[1] = qf[n][2 * i][1];
                    f[2] = qf[n][2 * i + 1][0];
                    f[3] = qf[n][2 * i + 1][1];
                }
            };
            float o[NR][KS][4];  // O^T: columns o_col(ds, kq, i), row 2 c + (i & 1)
            float mx[NR][2], sum[NR][2];
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                mx[n][0] = mx[n][1] = -INFINITY;
                sum[n][0] = sum[n][1] = 0.0f;
#pragma unroll
                for (int ds = 0; ds < KS; ++ds)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[n][ds][i] = 0.0f;
            }

            for (int j = t0; j < t1; ++j, advance()) {
                const int par = turn & 1, key0 = wk * 16, valid = min(kTile, sp.keys - j * kTile);
                const uint32_t sk = smem_addr(smem + st * C::STAGE), sv = sk + C::V_OFF;
                ok = ok && warp_wait(smem_addr(&sh.full_k[st]), par, abort);
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                if (key0 < valid) {
                    // ---- S^T = K Q^T: keys kq, kq + 8; rows 2 c, 2 c + 1 ----
                    float s[NR][4];
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
                    if constexpr (!Q8) {
#pragma unroll
                        for (int i = 0; i < KS / 2; ++i) {
                            uint32_t k0[4], k1[4];
                            load_k_rows<D>(sk, key0, 2 * i, lane, k0);
                            load_k_rows<D>(sk, key0, 2 * i + 1, lane, k1);
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
                    const bool masked = !sp.all_see(a, j * kTile + key0, 16);
                    uint32_t vis[NR][2];  // bit k: key0 + k visible to the row
                    bool above = false;
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) vis[n][e] = masked ? (p_of[n][e] < 0 ? 0u : seen_bits(a, sp, p_of[n][e], j * kTile + key0) & 0xffffu) : 0xffffu;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s[n][i] *= a.scale_log2;
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
                                for (int y = 4; y < 32; y <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, y));
                                m = fmaxf(m, mx[n][e]);
                                f[e] = m == -INFINITY ? 1.0f : ex2(mx[n][e] - m);
                                mx[n][e] = m;
                                sum[n][e] *= f[e];
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
                        if (Q8) {
                            sum[n][0] += s[n][0] + s[n][2];
                            sum[n][1] += s[n][1] + s[n][3];
                        }
                    }
                    // ---- O^T += V^T P^T ----
                    ok = warp_wait(smem_addr(&sh.full_v[st]), par, abort);
                    if (!ok) *abort = 1;
                    if constexpr (!Q8) {
                        if (masked) {
                            // 0 * inf would reach rows that do not see a value. So the values of keys that no row sees become 0, and
                            // those that are not finite of keys that some rows see (rare) go to those rows one by one. In shared
                            // memory, of which the warp's keys are its own, so that the products below have one form: with this among
                            // them a first masked tile waited for 4000 cycles of instructions.
                            uint32_t some = 0, every = 0xffffu;
#pragma unroll
                            for (int n = 0; n < NR; ++n)
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    if (p_of[n][e] >= 0) {
                                        some |= vis[n][e];
                                        every &= vis[n][e];
                                    }
                            some = __reduce_or_sync(0xffffffffu, some);
                            const bool differ = __reduce_and_sync(0xffffffffu, every) != some;
                            constexpr int U = D / 8;
                            uint8_t *const vt = smem + st * C::STAGE + C::V_OFF;
                            auto marks = [](const uint4 &v) {  // its values that are not finite, a bit each
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                                uint32_t m = 0;
#pragma unroll
                                for (int k = 0; k < 4; ++k) m |= ((w[k] & 0x7f80u) == 0x7f80u ? 1u : 0u) << 2 * k | ((w[k] & 0x7f800000u) == 0x7f800000u ? 2u : 0u) << 2 * k;
                                return m;
                            };
                            uint32_t bad = 0;
#pragma unroll 4
                            for (int i = lane; i < 16 * U; i += 32) {
                                uint4 *const at = (uint4 *)(vt + bf16_off<D>(key0 + i / U, i % U * 8));
                                if (!((some >> (i / U)) & 1u)) *at = make_uint4(0, 0, 0, 0);
                                else if (differ) bad |= marks(*at);
                            }
                            if (__any_sync(0xffffffffu, bad != 0)) {
#pragma unroll 1
                                for (int i = lane; i < 16 * U; i += 32) {
                                    uint4 *const at = (uint4 *)(vt + bf16_off<D>(key0 + i / U, i % U * 8));
                                    uint4 v = *at;
                                    const uint32_t m = marks(v);
                                    for (uint32_t lanes = __ballot_sync(0xffffffffu, m != 0); lanes; lanes &= lanes - 1) {
                                        const int from = __ffs(lanes) - 1, key = __shfl_sync(0xffffffffu, i, from) / U, unit = __shfl_sync(0xffffffffu, i, from) % U;
                                        const uint32_t w[4] = {__shfl_sync(0xffffffffu, v.x, from), __shfl_sync(0xffffffffu, v.y, from),
                                                               __shfl_sync(0xffffffffu, v.z, from), __shfl_sync(0xffffffffu, v.w, from)};
                                        const uint32_t of = __shfl_sync(0xffffffffu, m, from);
#pragma unroll
                                        for (int k = 0; k < 8; ++k) {
                                            if (kq != k || !((of >> k) & 1u)) continue;  // column 8 unit + k is this lane's
                                            const float y = __uint_as_float(k & 1 ? w[k / 2] & 0xffff0000u : w[k / 2] << 16);
#pragma unroll
                                            for (int ds = 0; ds < KS; ++ds)
#pragma unroll
                                                for (int n = 0; n < NR; ++n)
#pragma unroll
                                                    for (int x = 0; x < 4; ++x)
                                                        if (unit == 2 * ds + (x >> 1) && ((vis[n][x & 1] >> key) & 1u)) o[n][ds][x] += y;
                                        }
                                    }
                                    if (m & 1u) v.x &= 0xffff0000u;
                                    if (m & 2u) v.x &= 0xffffu;
                                    if (m & 4u) v.y &= 0xffff0000u;
                                    if (m & 8u) v.y &= 0xffffu;
                                    if (m & 16u) v.z &= 0xffff0000u;
                                    if (m & 32u) v.z &= 0xffffu;
                                    if (m & 64u) v.w &= 0xffff0000u;
                                    if (m & 128u) v.w &= 0xffffu;
                                    if (m) *at = v;
                                }
                            }
                            fence_proxy_async();  // the next tile comes here through the copy engine
                            __syncwarp();
                        }
                        uint32_t pr[NR][2];
#pragma unroll
                        for (int n = 0; n < NR; ++n) {
                            const uint32_t w0 = pack_bf16(s[n][0], s[n][1]), w1 = pack_bf16(s[n][2], s[n][3]);
                            sum[n][0] += __uint_as_float(w0 << 16) + __uint_as_float(w1 << 16);
                            sum[n][1] += __uint_as_float(w0 & 0xffff0000u) + __uint_as_float(w1 & 0xffff0000u);
                            pr[n][0] = movmatrix_trans(w0);
                            pr[n][1] = movmatrix_trans(w1);
                        }
#pragma unroll
                        for (int ds = 0; ds < KS; ++ds) {
                            uint32_t vf[4];
                            load_v_cols<D>(sv, key0, ds, lane, vf);
#pragma unroll
                            for (int n = 0; n < NR; ++n) mma_bf16(o[n][ds], vf, pr[n][0], pr[n][1]);
                        }
                    } else {
                        constexpr int G = D / 32;
                        const int kr[4] = {key0 + 2 * c, key0 + 2 * c + 1, key0 + 2 * c + 8, key0 + 2 * c + 9};
                        uint32_t sc[4][(G + 1) / 2];
#pragma unroll
                        for (int k = 0; k < 4; ++k) load_scales<G>(sv + T::SCALES + kr[k] * G * 2, sc[k]);
                        // the probabilities of row kq and keys kr, from the keys' lanes: as two bf16 each, which hold 16 bits of
                        // them, through the 16-bit transpose
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
                            uint32_t v0[4], v1[4], w[4];  // operands of the group's two 16-column steps
#pragma unroll
                            for (int k = 0; k < 4; ++k) w[k] = lds32(sv + q8_qs_off(kr[k], 32 * gr + 4 * kq, D));
                            int8x4_to_bf16(__byte_perm(w[0], w[1], 0x5140), v0[0], v0[1]);
                            int8x4_to_bf16(__byte_perm(w[2], w[3], 0x5140), v0[2], v0[3]);
                            int8x4_to_bf16(__byte_perm(w[0], w[1], 0x7362), v1[0], v1[1]);
                            int8x4_to_bf16(__byte_perm(w[2], w[3], 0x7362), v1[2], v1[3]);
                            float f[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) f[k] = scale_of(sc[k], gr);
#pragma unroll
                            for (int n = 0; n < NR; ++n) {
                                // (a key that the row does not see has p = 0, whatever its scale is)
                                float xs[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) xs[k] = masked && pt[n][k] == 0.0f ? 0.0f : pt[n][k] * f[k];
                                const uint32_t p0 = pack_bf16(xs[0], xs[1]), p1 = pack_bf16(xs[2], xs[3]);
                                // (an infinite scale has no remainder, and any finite number serves for it)
                                const uint32_t r0 = pack_bf16(fminf(xs[0] - __uint_as_float(p0 << 16), 3e38f), fminf(xs[1] - __uint_as_float(p0 & 0xffff0000u), 3e38f));
                                const uint32_t r1 = pack_bf16(fminf(xs[2] - __uint_as_float(p1 << 16), 3e38f), fminf(xs[3] - __uint_as_float(p1 & 0xffff0000u), 3e38f));
                                mma_bf16(o[n][2 * gr], v0, p0, p1);
                                mma_bf16(o[n][2 * gr + 1], v1, p0, p1);
                                mma_bf16(o[n][2 * gr], v0, r0, r1);
                                mma_bf16(o[n][2 * gr + 1], v1, r0, r1);
                            }
                        }
                    }
                } else {  // no key of this tile is the warp's: still stay in step with the stage
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
                    float l = sum[n][e];
#pragma unroll
                    for (int y = 4; y < 32; y <<= 1) l += __shfl_xor_sync(0xffffffffu, l, y);
                    if (kq == 0) sml[wk * C::ROWS + 8 * n + 2 * c + e] = make_float2(mx[n][e], l);
                }
            asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
            const bool joins = C::CLUSTERS && a.cluster > 1, whole = t0 == 0 && t1 == n_tiles && !joins;
            const long long slot = 2ll * blockIdx.x + (t0 == 0 ? 1 : 0);
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 8 * n + 2 * c + e;
                    float mt = -INFINITY, lt = 0.0f;
#pragma unroll
                    for (int w = 0; w < kKeyWarps; ++w) mt = fmaxf(mt, sml[w * C::ROWS + r].x);
                    const float mu = mt == -INFINITY ? 0.0f : mt;
#pragma unroll
                    for (int w = 0; w < kKeyWarps; ++w) {
                        const float2 ml = sml[w * C::ROWS + r];
                        lt += ml.y * ex2(ml.x - mu);
                    }
                    scale_o[n][e] = mx[n][e] == -INFINITY ? 0.0f : ex2(mx[n][e] - mu);
                    if (whole) scale_o[n][e] = lt == 0.0f ? 0.0f : scale_o[n][e] / lt;
                    if (wk != 0 || kq != 0 || r >= rows || whole) continue;
                    if (joins) {
                        const uint32_t at = smem_addr(part_ml + rank * C::ROWS + r);
                        for (int k = 0; k < a.cluster; ++k) stc128(mapa_shared(at, k), make_float4(mt, lt, 0.0f, 0.0f));
                    } else {
                        a.ws_ml[slot * C::ROWS + r] = make_float4(mt, lt, 0.0f, 0.0f);
                    }
                }
            const int share = (rows * (D / 4) + a.cluster - 1) / a.cluster;  // float4 outputs that a CTA of the cluster writes
            constexpr int XC = C::X_COLS, ROUNDS = D / XC, Q4 = XC / 4;
#pragma unroll
            for (int cc = 0; cc < ROUNDS; ++cc) {
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int d2 = 0; d2 < XC / 16; ++d2)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int ds = cc * (XC / 16) + d2, r = 8 * n + 2 * c + (i & 1), col = o_col<Q8>(ds, kq, i) - cc * XC;
                            // a warp without a key for the row has nothing (not 0 * its garbage)
                            const float f = scale_o[n][i & 1];
                            xb[(wk * C::ROWS + r) * XC + ((col + 4 * r) & (XC - 1))] = f == 0.0f ? 0.0f : o[n][ds][i] * f;
                        }
                asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
                for (int i = threadIdx.x; i < rows * Q4; i += C::NC) {
                    const int r = i / Q4, col = (i - r * Q4) * 4;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < kKeyWarps; ++w) {
                        const float4 y = *(const float4 *)&xb[(w * C::ROWS + r) * XC + ((col + 4 * r) & (XC - 1))];
                        v.x += y.x;
                        v.y += y.y;
                        v.z += y.z;
                        v.w += y.w;
                    }
                    if (joins) {  // to the CTA that writes it
                        const int item = r * (D / 4) + (cc * XC + col) / 4, to = item / share;
                        stc128(mapa_shared(smem_addr(part_o + rank * share + item - to * share), to), v);
                    } else if (!whole) {
                        *(float4 *)(a.ws_o + (slot * C::ROWS + r) * D + cc * XC + col) = v;
                    } else {
                        const int t = row_token(a, r);
                        *(uint2 *)(a.out + ((src_row + t) * a.q_heads + g * a.group + r - t * a.group) * D + cc * XC + col) =
                            make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
                    }
                }
                // (the next unit's end has a barrier before these are written again)
                if (cc + 1 < ROUNDS) asm volatile("bar.sync 1, %0;" ::"n"(C::NC) : "memory");
            }
        }
        if constexpr (C::CLUSTERS)
            if (a.cluster > 1) {
                // out = sum_k 2^(m_k - m) o_k / sum_k 2^(m_k - m) l_k over the cluster's CTAs k
                __syncwarp();
                if (warp == kKeyWarps) cluster_wait();
                cluster_sync();  // everyone's parts are here
                const int share = (rows * (D / 4) + a.cluster - 1) / a.cluster;
                for (int i = threadIdx.x; i < share && rank * share + i < rows * (D / 4); i += C::THREADS) {
                    const int item = rank * share + i, r = item / (D / 4), col = (item - r * (D / 4)) * 4;
                    float m = -INFINITY, l = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int k = 0; k < a.cluster; ++k) m = fmaxf(m, part_ml[k * C::ROWS + r].x);
                    for (int k = 0; k < a.cluster; ++k) {
                        const float4 ml = part_ml[k * C::ROWS + r], y = part_o[k * share + i];
                        const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m);
                        l += f * ml.y;
                        if (f == 0.0f) continue;  // (a part that saw nothing for the row)
                        v.x = fmaf(y.x, f, v.x);
                        v.y = fmaf(y.y, f, v.y);
                        v.z = fmaf(y.z, f, v.z);
                        v.w = fmaf(y.w, f, v.w);
                    }
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    const int t = row_token(a, r);
                    *(uint2 *)(a.out + ((src_row + t) * a.q_heads + g * a.group + r - t * a.group) * D + col) =
                        make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
                }
            }
        if (!a.split) break;
        x += t1 - t0;
    }
    if (!ok && lane == 0) report_error(a.pool.status, DEV_ERR_TIMEOUT, blockIdx.x, warp, 16);
    if (warp == kKeyWarps && !ok && lane == 0) {
        // leave no copy writing this CTA's shared memory: the last uses of every stage that were issued
        for (int i = 0; i < NST; ++i) {
            mbar_wait_drain(smem_addr(&sh.full_k[i]), 0, kWait / 64);
            mbar_wait_drain(smem_addr(&sh.full_k[i]), 1, kWait / 64);
            mbar_wait_drain(smem_addr(&sh.full_v[i]), 0, kWait / 64);
            mbar_wait_drain(smem_addr(&sh.full_v[i]), 1, kWait / 64);
        }
    }
}

// Rows of units that several CTAs took parts of: out = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c, a warp for each row. Lanes look
// at 32 parts' maxima and sums at once, so that the parts' rows are read without waiting for one another.
constexpr int kMergeWarps = 8;
constexpr int kMaxRangeRequests = 4096;  // (their places take 16 KB of the tile kernel's shared memory)

template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32) window_merge_kernel(const WindowArgs a, int unit_rows) {
    const int lane = threadIdx.x & 31, blocks = unit_rows / kMergeWarps;
    const int unit = blockIdx.x / blocks, r = (blockIdx.x - unit * blocks) * kMergeWarps + (threadIdx.x >> 5);
    // a unit (rows kernel), or the one that CTA `unit` began (tile kernel)
    const int hk = a.pool.kv_heads;
    int flat = unit / hk, g = unit - flat * hk;
    int2 part = make_int2(unit, 0);
    grid_wait();
    if (a.cuts) {
        const int4 cut = a.cuts[unit];
        if (cut.w == 0) return;
        flat = cut.x;
        g = cut.y;
        part.y = cut.z;
    }
    const int b = flat / a.row_tiles, row = (flat - b * a.row_tiles) * unit_rows + r;
    const WinReq rq = load_win_req(a, b, false);
    if (rq.seq < 0 || row >= rq.n * a.group) return;
    if (!a.cuts) part = a.parts[unit];
    if (part.x == part.y) return;
    constexpr int PER = (D + 127) / 128;  // float4 of a lane
    auto part_row = [&](int c) { return (2ll * c + (c == part.x ? 1 : 0)) * unit_rows + r; };
    float m = -INFINITY;
    for (int c = part.x + lane; c <= part.y; c += 32) m = fmaxf(m, a.ws_ml[part_row(c)].x);
#pragma unroll
    for (int y = 1; y < 32; y <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, y));
    float l = 0.0f;
    float4 o[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c0 = part.x; c0 <= part.y; c0 += 32) {
        float f = 0.0f;
        if (c0 + lane <= part.y) {
            const float4 ml = a.ws_ml[part_row(c0 + lane)];
            f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m);
            l += f * ml.y;
        }
        const int n = min(32, part.y + 1 - c0);
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
            const float fk = __shfl_sync(0xffffffffu, f, k);
            const float4 *src = (const float4 *)(a.ws_o + part_row(c0 + k) * D);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (lane + 32 * i < D / 4 && fk != 0.0f) {  // (a part that saw nothing for the row: its output may be anything)
                    const float4 v = src[lane + 32 * i];
                    o[i].x = fmaf(v.x, fk, o[i].x);
                    o[i].y = fmaf(v.y, fk, o[i].y);
                    o[i].z = fmaf(v.z, fk, o[i].z);
                    o[i].w = fmaf(v.w, fk, o[i].w);
                }
        }
    }
#pragma unroll
    for (int y = 1; y < 32; y <<= 1) l += __shfl_xor_sync(0xffffffffu, l, y);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int t = row_token(a, row);
    uint2 *to = (uint2 *)(a.out + (((int64_t)a.src_row[b] + t) * a.q_heads + g * a.group + row - t * a.group) * D);
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < D / 4) to[lane + 32 * i] = make_uint2(pack_bf16(o[i].x * inv, o[i].y * inv), pack_bf16(o[i].z * inv, o[i].w * inv));
}

// ---- host side ----
bool few_rows(int rows) { return rows <= kFewRows; }
int unit_rows(const PoolView &p, int rows) { return few_rows(rows) ? (rows <= 8 ? 8 : 16) : window_tile_rows(p.head_dim); }
int full_grid(const PoolView &p, int rows, int sms) {
    return sms * (few_rows(rows) ? few_ctas(p.head_dim, p.dtype == EKV_DTYPE_Q8_0, rows <= 8 ? 1 : 2) : 1);
}

struct WsLayout {
    size_t ml, o, total;
};
WsLayout ws_layout(const PoolView &p, int n_batch, int rows, int sms) {
    const size_t ur = (size_t)unit_rows(p, rows), slots = 2 * (size_t)full_grid(p, rows, sms) * ur, row_tiles = ((size_t)rows + ur - 1) / ur;
    WsLayout w;
    const size_t joins = few_rows(rows) ? (size_t)n_batch * p.kv_heads * row_tiles * sizeof(int2) : slots / ur / 2 * sizeof(int4);
    w.ml = (joins + 255) / 256 * 256;
    w.o = w.ml + slots * sizeof(float4);
    w.total = w.o + slots * p.head_dim * sizeof(float);
    return w;
}

template <int D, bool Q8, int NR>
int rows_smem() {
    static std::atomic<uint64_t> done{0};
    return allow_smem(window_rows_kernel<D, Q8, NR>, FCfg<D, Q8, NR>::SMEM, done);
}

template <int D, bool Q8, int NR>
int launch_rows(const WindowArgs &a, int grid, cudaStream_t s) {
    using C = FCfg<D, Q8, NR>;
    if (const int rc = rows_smem<D, Q8, NR>()) return rc;
    return launch_clusters_after(a.cluster, window_rows_kernel<D, Q8, NR>, grid, C::THREADS, C::SMEM, s, a);
}

// Clusters of 2^(i + 1) CTAs that run at the same time on the current device (asked once: it depends on how many SMs each part of the
// device has; 0 where that cannot be asked).
template <int D, bool Q8, int NR>
int rows_clusters(int i) {
    using C = FCfg<D, Q8, NR>;
    static std::atomic<int> known[64][3];  // 1 + their number
    int dev = 0, n = 0;
    if (!C::CLUSTERS || cudaGetDevice(&dev) != cudaSuccess || dev >= 64 || rows_smem<D, Q8, NR>()) return 0;
    std::atomic<int> &k = known[dev][i];
    if (const int have = k.load(std::memory_order_relaxed)) return have - 1;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(2u << i);
    c.blockDim = dim3((unsigned)C::THREADS);
    c.dynamicSmemBytes = C::SMEM;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2u << i;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, window_rows_kernel<D, Q8, NR>, &c) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    k.store(n + 1, std::memory_order_relaxed);
    return n;
}

// f with head_dim, 8-bit pages, and groups of eight rows (0: the tile kernel) as types.
template <class F>
int with_form(const PoolView &p, int rows, F f) {
    const bool q8 = p.dtype == EKV_DTYPE_Q8_0;
    auto dim = [&](auto d) {
        using D = decltype(d);
        using T = std::true_type;
        using N = std::false_type;
        if (!few_rows(rows)) return f(d, N{}, std::integral_constant<int, 0>{});
        if (rows <= 8) return q8 ? f(D{}, T{}, std::integral_constant<int, 1>{}) : f(D{}, N{}, std::integral_constant<int, 1>{});
        return q8 ? f(D{}, T{}, std::integral_constant<int, 2>{}) : f(D{}, N{}, std::integral_constant<int, 2>{});
    };
    switch (p.head_dim) {
        case 64: return dim(std::integral_constant<int, 64>{});
        case 128: return dim(std::integral_constant<int, 128>{});
        case 256: return dim(std::integral_constant<int, 256>{});
        default: return EKV_ERR_UNSUPPORTED;
    }
}

}  // namespace

size_t window_workspace(const PoolView &p, int n_batch, int max_rows, int q_heads, int sms) {
    return ws_layout(p, n_batch, max_rows * (q_heads / p.kv_heads), sms).total;
}

int launch_window_attention(WindowArgs a, int max_len, void *ws, size_t ws_bytes, int sms, cudaStream_t s) {
    const int rows = a.max_rows * a.group, ur = unit_rows(a.pool, rows), keys = few_rows(rows) ? kTile : window_tile_keys();
    a.row_tiles = (rows + ur - 1) / ur;
    const int64_t units = (int64_t)a.n_batch * a.row_tiles * a.pool.kv_heads;
    if (units * (ur / kMergeWarps) > INT32_MAX) return EKV_ERR_INVALID_ARG;
    const int full = full_grid(a.pool, rows, sms);
    const WsLayout w = ws_layout(a.pool, a.n_batch, rows, sms);
    // a unit's tiles at most: its tokens, the window before the first of them, the first tokens
    const int64_t tokens = std::min<int64_t>(a.max_rows, (ur + a.group - 1) / a.group + 1);
    auto tiles = [&](int64_t len) { return (std::min<int64_t>(len, (int64_t)a.window + tokens + a.sinks) + 16 + keys - 1) / keys; };
    const int64_t unit_tiles = tiles(max_len), most_tiles = tiles((int64_t)a.pool.max_blocks_per_seq * a.pool.block_tokens) + 1;
    const bool can_split = ws != nullptr && ws_bytes >= w.total && units * (most_tiles + kWindowUnitCost) < INT32_MAX;
    a.split = 0;
    a.cluster = 1;
    int64_t grid;
    if (few_rows(rows)) {
        // A cluster of CTAs per unit, or equal ranges of all tiles and a join; times in tiles. A call costs `fixed` beside its
        // tiles, the join `worth`, which grows with the parts of a unit: 64 requests of 17 tiles of head_dim 256, bf16 22.1 us with clusters of 2, 33.1 with 4 (which run in two
        // turns), 29.9 with a join; 16 of them 13.4 with clusters of 4, 21.7 with 8 (two turns) and with a join. 8-bit pages: 32 requests
        // 37.1, 23.7, 17.9, 15.3 with 1, 2, 4, 8, 24.1 with a join; 128 of 17 tiles 32.9 with 2, 39.9 with 1, 39.1 with a join; one of 65 tiles
        // 22.6 with 8, 33.4 with a join of 65 parts. 128 units of 129 tiles of head_dim 128, bf16: 84 with clusters of 2, 92 with a join.
        const bool q8 = a.pool.dtype == EKV_DTYPE_Q8_0;
        const int64_t even = (units * unit_tiles + full - 1) / full, parts = (unit_tiles + even - 1) / std::max<int64_t>(1, even);
        const int64_t fixed = q8 ? 4 : 8, worth = q8 ? std::max<int64_t>(7, 5 + parts / 7) : std::max<int64_t>(10, 8 + parts / 4);
        int64_t best = (units + full - 1) / full * (fixed + unit_tiles);
        for (int i = 0; i < 3 && (2 << i) <= unit_tiles; ++i) {
            const int c = 2 << i;
            const int64_t fit = with_form(a.pool, rows, [&](auto d, auto q, auto nr) {
                if constexpr (decltype(nr)::value > 0) return rows_clusters<decltype(d)::value, decltype(q)::value, decltype(nr)::value>(i);
                else return 0;
            });
            if (fit <= 0) break;
            const int64_t cost = (units + fit - 1) / fit * (fixed + (unit_tiles + c - 1) / c);
            if (cost < best) {
                best = cost;
                a.cluster = c;
            }
        }
        if (can_split && fixed + even + worth < best) {
            a.split = kCutUnits;
            a.cluster = 1;
        }
        grid = a.split ? std::min<int64_t>(full, units * unit_tiles) : units * a.cluster;
    } else {
        // Up to four units a CTA: whole ones, the longest first. More: ranges of whole units, which know how many rows the requests have
        // (32 requests of 100 to 500 rows: 197 us, the longest first 262). Cut ranges where the longest CTA would have more than 40 tiles
        // above the even share, or 16 where none has two units: cutting costs 25 us, for the parts' way through memory and the join.
        // Whole in order, whole by ranges, cut: 64 requests of 77 rows, a window of 300 (1.7 units a CTA): 25, 35, 40 us; a prompt of 4096
        // tokens (3.5) 166, 208, 197; 3 prompts of up to 2048 (5.2) 126, 99, 112; 8 of up to 4096, a window of 1024 (28) 680, 633, 655;
        // 5 requests of 200 rows, a window of 2000 (0.3) 46, 49, 26; one prompt of 16384 (14) 2419, 2568, 2383.
        const int64_t cost = unit_tiles + kWindowUnitCost;
        const bool ranges = a.n_batch <= kMaxRangeRequests && units * (most_tiles + kWindowUnitCost) < INT32_MAX;
        const int64_t over = ((units + full - 1) / full * full - units) * cost / full;
        if (ranges && can_split && over > (units > full ? 40 : 16)) a.split = kCutUnits;
        else if (ranges && units > 4 * full) a.split = kWholeUnits;
        grid = std::min<int64_t>(full, a.split == kCutUnits ? units * cost : units);
    }
    if (a.split == kCutUnits) {
        a.parts = (int2 *)ws;
        a.cuts = few_rows(rows) ? nullptr : (int4 *)ws;
        a.ws_ml = (float4 *)((uint8_t *)ws + w.ml);
        a.ws_o = (float *)((uint8_t *)ws + w.o);
    }
    if (grid > INT32_MAX) return EKV_ERR_INVALID_ARG;
    return with_form(a.pool, rows, [&](auto d, auto q, auto nr) {
        constexpr int D = decltype(d)::value, NR = decltype(nr)::value;
        int rc;
        if constexpr (NR > 0) rc = launch_rows<D, decltype(q)::value, NR>(a, (int)grid, s);
        else rc = launch_window_tile(a, (int)grid, s);
        if (rc || a.split != kCutUnits) return rc;
        const int n_units = a.cuts ? (int)grid : (int)units;
        return launch_after(window_merge_kernel<D>, n_units * (ur / kMergeWarps), kMergeWarps * 32, 0, s, a, ur);
    });
}

}  // namespace ekv
