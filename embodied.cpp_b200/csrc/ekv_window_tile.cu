// ekv_window_tile.cu -- windowed attention of many rows per KV head (prompts, chunks) on tcgen05.
//
// out = sum_k p_k v_k / sum_k p_k with p_k = exp(scale q.k - m) over the keys a row sees (ekv_window.cuh), m a running reference that
// moves only when a score is 2^8 above it. S = Q K^T with both operands in shared memory and S in tensor memory, P in 16 bits over
// S's own columns, O += P V with P read from tensor memory. P is rounded to bf16 (bf16 pages) and the row divided by the sum of the
// rounded ones; over 8-bit pages operands are f16 (a value's int8 times its scale keeps 11 bits, P too).
#include "ekv_window.cuh"

namespace ekv {
namespace {

using namespace decode;
using namespace sm100;
using namespace window;

constexpr int kTileRows = 128;  // rows of a row tile: the lanes of tensor memory

// head_dim 64 and 128: two row tiles (slots) of a KV head share an SM and each K/V tile of 128 keys. While one slot's exponentials
// run, the other's products do. head_dim 256: one row tile, 64 keys, two S tiles, as two outputs do not fit the tensor memory.
template <int D, bool Q8>
struct WCfg {
    static constexpr int RT = D > 128 ? 1 : 2;
    static constexpr int BN = D > 128 ? 64 : 128;     // keys per tile
    static constexpr int NSB = D > 128 ? 2 : 1;       // S tiles of a row tile
    static constexpr int NS = D == 64 ? 4 : 2;        // K and V stages
    static constexpr int KPW = BN / 2;                // keys of a tile per softmax warp: two warps share 32 rows
    static constexpr uint32_t SBO = 16 * D, LAYOUT = 2;
    static constexpr int KV_BYTES = BN * D * 2, Q_BYTES = kTileRows * D * 2;
    static constexpr int RK = 8192 / D;               // Q8: keys of a piece of blocks as they are stored
    static constexpr int NR = 3, RAW = RK * D + RK * (D / 32) * 2;
    static constexpr int S_COL = 0, O_COL = BN * NSB, SLOT_COLS = 256, COLS = 512;
    static constexpr int OFF_K = RT * Q_BYTES, OFF_V = OFF_K + NS * KV_BYTES, OFF_RAW = OFF_V + NS * KV_BYTES;
    static constexpr int OFF_SH = OFF_RAW + (Q8 ? (NR * RAW + 1023) / 1024 * 1024 : 0);
    static constexpr int SHARED = 4096 + RT * 2 * kTileRows * 4, SMEM = OFF_SH + SHARED + 1024;
    static constexpr int ROW_WARPS = 8 * RT, MMA_WARP = ROW_WARPS, FEED_WARP = MMA_WARP + RT;
    // bf16: K's feeder, V's feeder, and a warp that looks at V; Q8: one feeder, and converters
    static constexpr int SCRUB_WARP = FEED_WARP + 2, CONV_WARP = FEED_WARP + 1, CONV_WARPS = RT == 1 ? 8 : 4;
    static constexpr int THREADS = (Q8 ? CONV_WARP + CONV_WARPS : SCRUB_WARP + 1) * 32;
    static_assert(O_COL + D <= (RT == 2 ? SLOT_COLS : COLS) && SMEM <= 232448, "tensor memory, shared memory");
};

constexpr int kBadTiles = 10;  // a unit has at most ten tiles that only some of its rows see: three of 128 keys around 256 tokens'
                               // own slots, three around the window's end, two around the first tokens, and the last one
constexpr int kBadUnits = 8;   // V is looked at no more than the stages' tiles ahead of the rows

struct WShared {
    uint64_t full_k[4], full_v[4];       // K, V of the stage are there
    uint64_t raw_full[3], raw_empty[3];  // Q8: a piece has landed; is converted
    uint64_t s_full[2][4];               // [slot][stage] S done
    uint64_t v_free[4];                  // both slots' P V done, and (bf16) the tile looked at
    uint64_t p_full[2][2];               // [slot][S tile] P written
    uint64_t q_ready[2], o_done[2], drained[2];
    uint64_t v_clean[4];                 // V of a tile that only some rows see holds finite values
    uint32_t bad[kBadUnits][kBadTiles][4];  // [unit % kBadUnits] its keys that did not
    int bad_key[kBadUnits][kBadTiles], n_bad[kBadUnits];
    uint32_t tmem;
    int abort;
    RangeScratch range;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Two warps that share 32 rows (64 threads of a named barrier). Both take the same way through these whatever else fails, so that
// neither is left waiting.
__device__ __forceinline__ bool pair_any(int id, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)x), "r"(id)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void pair_sync(int id) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory"); }

// Where a unit is, and its keys.
struct Unit {
    int b, g, row0, rows_all;  // request, KV head, first row, the request's rows
    WinReq rq;
};

// The blocks' int8 rows as f16 values, rounded once; rows past `valid` are zero. Scales that leave the f16 range with them are
// reported, their values 0.
template <int D, int ROWS, int THREADS>
__device__ __forceinline__ bool convert_piece(const uint8_t *raw, uint8_t *dst, int row0, int valid, int thread) {
    constexpr int U = D / 16;
    bool fits = true;
#pragma unroll 2
    for (int e = thread; e < ROWS * U; e += THREADS) {
        // four 16-byte columns and two rows in every eight lanes, which then write to eight different columns of the swizzled rows
        const int rest = e >> 3, u = (rest % (U / 4)) * 4 + (e & 3), row = rest / (U / 4) * 2 + ((e >> 2) & 1);
        uint32_t out[8] = {};
        if (row < valid) {
            const uint4 v = *(const uint4 *)(raw + q8_qs_off(row, 16 * u, D));
            const uint16_t bits = *(const uint16_t *)(raw + ROWS * D + (row * (D / 32) + (u >> 1)) * 2);
            const bool ok = fabsf(f16_bits_to_f32(bits)) <= 515.0f;
            fits = fits && ok;
            const __half2 d = __half2half2(__ushort_as_half(ok ? bits : (uint16_t)0)), base = __half2half2(__ushort_as_half(0x6480));  // 1152
            const uint32_t w[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    // byte 0x64 above a byte u is the f16 1024 + u, and u = x + 128
                    const uint32_t m = __byte_perm(w[i], 0x64646464u, k ? 0x4342 : 0x4140);
                    const __half2 x = __hmul2(__hsub2(*(const __half2 *)&m, base), d);
                    out[2 * i + k] = *(const uint32_t *)&x;
                }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
            *(uint4 *)(dst + bf16_off<D>(row0 + row, 16 * u + 8 * k)) = make_uint4(out[4 * k], out[4 * k + 1], out[4 * k + 2], out[4 * k + 3]);
    }
    return fits;
}

template <int D, bool Q8>
__global__ void __launch_bounds__(WCfg<D, Q8>::THREADS, 1) window_tile_kernel(const WindowArgs a) {
    using C = WCfg<D, Q8>;
    constexpr int BN = C::BN, NS = C::NS, NSB = C::NSB, RT = C::RT, ROWS = RT * kTileRows, KPW = C::KPW;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    WShared &sh = *(WShared *)(smem + C::OFF_SH);
    static_assert(sizeof(WShared) <= 4096, "barrier block");
    float *const s_x = (float *)(smem + C::OFF_SH + 4096);  // [slot][warp of the pair][row]
    volatile int *abort = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = a.pool.kv_heads;

    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(smem_addr(&sh.full_k[i]), Q8 ? C::CONV_WARPS : 1);
            mbar_init(smem_addr(&sh.full_v[i]), Q8 ? C::CONV_WARPS : 1);
            mbar_init(smem_addr(&sh.v_free[i]), Q8 ? RT : RT + 1);
            mbar_init(smem_addr(&sh.v_clean[i]), 1);
            for (int k = 0; k < RT; ++k) mbar_init(smem_addr(&sh.s_full[k][i]), 1);
        }
        for (int k = 0; k < RT; ++k) {
            for (int i = 0; i < NSB; ++i) mbar_init(smem_addr(&sh.p_full[k][i]), 8);
            mbar_init(smem_addr(&sh.q_ready[k]), 8);
            mbar_init(smem_addr(&sh.o_done[k]), 1);
            mbar_init(smem_addr(&sh.drained[k]), 1);
        }
        for (int i = 0; Q8 && i < C::NR; ++i) {
            mbar_init(smem_addr(&sh.raw_full[i]), 1);
            mbar_init(smem_addr(&sh.raw_empty[i]), C::CONV_WARPS);
        }
        sh.abort = 0;
        mbar_init_fence();
    }
    // request b's row tile t, without its tiles (units in the flat order of a split: request, row tile, KV head)
    const int n_tiles_rt = a.row_tiles;
    auto tiles_of = [&](const WinReq &r, int rt) {
        const int row0 = rt * ROWS, rows_all = r.n * a.group;
        if (row0 >= rows_all) return 0;
        const Span sp(a, r, row_token(a, row0), last_token(a, row0, ROWS, r.n));
        return max(1, (sp.keys + BN - 1) / BN);
    };
    grid_wait();
    // (tensor memory between the two launch points: ekv_tree_tile.cu says why)
    if (warp == C::MMA_WARP) tmem_alloc(smem_addr(&sh.tmem), C::COLS);
    tc_fence_before();
    Range rg;
    rg.b = 0;
    rg.base = rg.lo = rg.hi = rg.total = 0;
    rg.ctas = 0;
    if (a.split) {
        rg = find_range<C::THREADS>(
            a.n_batch * n_tiles_rt, hk, sh.range,
            [&](int i) {
                const WinReq r = load_win_req(a, i / n_tiles_rt, false);
                return Req{0, tiles_of(r, i % n_tiles_rt), 0};
            },
            [](const Req &r) { return r.n_prefix; });
    } else {
        __syncthreads();
    }
    tc_fence_after();
    const uint32_t tmem = sh.tmem;  // (there is a barrier in either branch)
    grid_launch_next();

    // ---- the units of this CTA, in the same order in every warp ----
    // split: the tiles [rg.lo, rg.hi); else whole units, the longest (a request's last rows) first, back and forth over the CTAs
    const int n_flat = a.n_batch * n_tiles_rt;
    int flat = rg.b, round = 0;
    uint32_t base = rg.base, x = rg.lo;
    Unit u;
    int t0 = 0, t1 = 0, n_tiles = 0;
    // flat: request * row tiles + row tile (split), or the place in the order of units
    auto next_unit = [&]() -> bool {
        if (a.split) {
            for (; x < rg.hi && flat < n_flat; ++flat) {
                u.b = flat / n_tiles_rt;
                const int rt = flat - u.b * n_tiles_rt;
                u.rq = load_win_req(a, u.b, false);
                n_tiles = tiles_of(u.rq, rt);
                const uint32_t span = (uint32_t)n_tiles * hk;
                if (x >= base + span) {
                    base += span;
                    continue;
                }
                u.g = (int)((x - base) / (uint32_t)n_tiles);
                t0 = (int)(x - base) - u.g * n_tiles;
                t1 = min(n_tiles, t0 + (int)(rg.hi - x));
                u.row0 = rt * ROWS;
                u.rows_all = u.rq.n * a.group;
                x += t1 - t0;
                return true;
            }
            return false;
        }
        const long long all = (long long)n_flat * hk;
        for (;;) {
            const long long at = (long long)round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
            if ((long long)round * gridDim.x >= all) return false;
            ++round;
            if (at >= all) continue;
            const int rest = (int)(at / hk), rt = n_tiles_rt - 1 - rest / a.n_batch;
            u.g = (int)(at - (long long)rest * hk);
            u.b = rest - rest / a.n_batch * a.n_batch;
            u.rq = load_win_req(a, u.b, warp == 0 && rt == 0 && u.g == 0 && lane == 0);
            n_tiles = tiles_of(u.rq, rt);
            if (n_tiles == 0) continue;
            u.row0 = rt * ROWS;
            u.rows_all = u.rq.n * a.group;
            t0 = 0;
            t1 = n_tiles;
            return true;
        }
    };
    if (a.split && blockIdx.x == 0)  // (whoever has a request's unit does not report it: the first CTA looks at all)
        for (int b = threadIdx.x; b < a.n_batch; b += C::THREADS) load_win_req(a, b, true);

    bool ok = true, fits = true;
    int it = 0;       // tiles of this CTA so far
    int unit_no = 0;  // units so far
    int raw_it = 0;   // Q8: pieces so far
    int live_it[1] = {0};  // tiles so far that this slot had rows for (products and softmax)
    int live_units = 0;
    uint32_t clean_phase = 0;  // v_clean, a bit per stage

    while (next_unit()) {
        const int n = t1 - t0;
        const Span sp(a, u.rq, row_token(a, u.row0), last_token(a, u.row0, ROWS, u.rq.n));
        const int rows_here = min(ROWS, u.rows_all - u.row0);
        auto unit_sees = [&](int j) { return sp.all_see(a, j * BN, BN); };

        if (warp >= C::FEED_WARP && warp < (Q8 ? C::CONV_WARP : C::SCRUB_WARP)) {
            // ---- feeders ----
            auto want = [](int, int) {};
            auto block = [&](int e) { return lookup_block(a.pool, u.rq.seq, e); };
            const int64_t v_from_k = (int64_t)hk * a.pool.tile_bytes;
            if constexpr (!Q8) {
                const bool is_v = warp != C::FEED_WARP;
                Run next = find_run<BN>(a, sp, u.g, t0 * BN, lane, want, block);
                for (int j = t0; j < t1; ++j, ++it) {
                    const int st = it % NS, par = (it / NS) & 1;
                    const Run r = next;
                    if (j + 1 < t1) next = find_run<BN>(a, sp, u.g, (j + 1) * BN, lane, want, block);
                    if (it >= NS) {
                        if (is_v) ok = ok && warp_wait(smem_addr(&sh.v_free[st]), par ^ 1, abort);
#pragma unroll
                        for (int k = 0; k < RT; ++k)
                            if (!is_v) ok = ok && warp_wait(smem_addr(&sh.s_full[k][st]), par ^ 1, abort);
                    }
                    if (!ok) {
                        *abort = 1;
                        continue;
                    }
                    const uint32_t dst = smem_addr(smem + (is_v ? C::OFF_V : C::OFF_K) + st * C::KV_BYTES);
                    const uint32_t bar = smem_addr(is_v ? &sh.full_v[st] : &sh.full_k[st]);
                    const uint32_t bytes = r.src ? (uint32_t)(r.n * 2 * D) : 0u, all = __reduce_add_sync(0xffffffffu, bytes);
                    if (lane == 0) mbar_arrive_expect_tx(bar, all);
                    __syncwarp();
                    if (r.src) bulk_g2s(dst + r.row * 2 * D, r.src + (is_v ? v_from_k : 0) + r.rib * 2 * D, bytes, bar);
                }
            } else {
                constexpr int PIECES = BN / C::RK;  // of K, then of V
                for (int j = t0; j < t1; ++j)
                    for (int pc = 0; pc < 2 * PIECES; ++pc, ++raw_it) {
                        const bool is_v = pc >= PIECES;
                        const int key = j * BN + (pc - (is_v ? PIECES : 0)) * C::RK, rs = raw_it % C::NR;
                        const Run r = find_run<C::RK>(a, sp, u.g, key, lane, want, block);
                        if (raw_it >= C::NR) ok = ok && warp_wait(smem_addr(&sh.raw_empty[rs]), (raw_it / C::NR - 1) & 1, abort);
                        if (!ok) {
                            *abort = 1;
                            continue;
                        }
                        const uint32_t dst = smem_addr(smem + C::OFF_RAW + rs * C::RAW), bar = smem_addr(&sh.raw_full[rs]);
                        const uint32_t bytes = r.src ? (uint32_t)(r.n * (D + D / 16)) : 0u, all = __reduce_add_sync(0xffffffffu, bytes);
                        if (lane == 0) mbar_arrive_expect_tx(bar, all);
                        __syncwarp();
                        if (!r.src) continue;
                        const uint8_t *src = r.src + (is_v ? v_from_k : 0);
                        bulk_g2s(dst + r.row * D, src + r.rib * D, (uint32_t)(r.n * D), bar);
                        bulk_g2s(dst + C::RK * D + r.row * (D / 16), src + (int64_t)a.pool.block_tokens * D + r.rib * (D / 16),
                                 (uint32_t)(r.n * (D / 16)), bar);
                    }
            }
        } else if (Q8 && warp >= C::CONV_WARP) {
            // ---- converters ----
            constexpr int PIECES = BN / C::RK;
            const int thread = threadIdx.x - C::CONV_WARP * 32;
            for (int j = t0; j < t1; ++j, ++it) {
                const int st = it % NS, par = (it / NS) & 1;
                for (int pc = 0; pc < 2 * PIECES; ++pc, ++raw_it) {
                    const bool is_v = pc >= PIECES;
                    const int row0 = (pc - (is_v ? PIECES : 0)) * C::RK, rs = raw_it % C::NR;
                    if (row0 == 0 && it >= NS) {  // the stage is free
                        if (is_v) ok = ok && warp_wait(smem_addr(&sh.v_free[st]), par ^ 1, abort);
#pragma unroll
                        for (int k = 0; k < RT; ++k)
                            if (!is_v) ok = ok && warp_wait(smem_addr(&sh.s_full[k][st]), par ^ 1, abort);
                    }
                    ok = ok && warp_wait(smem_addr(&sh.raw_full[rs]), (raw_it / C::NR) & 1, abort);
                    if (!ok) {
                        *abort = 1;
                        continue;
                    }
                    fits &= convert_piece<D, C::RK, C::CONV_WARPS * 32>(smem + C::OFF_RAW + rs * C::RAW, smem + (is_v ? C::OFF_V : C::OFF_K) + st * C::KV_BYTES,
                                                                       row0, sp.keys - j * BN - row0, thread);
                    fence_proxy_async();  // read by the tensor core; the piece's next contents come through the copy engine
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(smem_addr(&sh.raw_empty[rs]));
                        if (row0 + C::RK == BN) mbar_arrive(smem_addr(is_v ? &sh.full_v[st] : &sh.full_k[st]));
                    }
                }
            }
        } else if (!Q8 && warp == C::SCRUB_WARP) {
            // ---- values that are not finite leave the tiles that only some rows see: 0 * inf would reach the others ----
            const int ub = unit_no % kBadUnits;
            if (lane == 0) sh.n_bad[ub] = 0;
            for (int j = t0; j < t1; ++j, ++it) {
                // (every tile is waited for and let go, whether it is looked at or not: a barrier's parity tells two phases apart)
                const int st = it % NS;
                ok = ok && warp_wait(smem_addr(&sh.full_v[st]), (it / NS) & 1, abort);
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                if (unit_sees(j)) {
                    if (lane == 0) mbar_arrive(smem_addr(&sh.v_free[st]));
                    continue;
                }
                uint8_t *vt = smem + C::OFF_V + st * C::KV_BYTES;
                constexpr int U = D / 8;
                const int valid = min(BN, sp.keys - j * BN);
                uint32_t bad[4] = {};
                for (int e = lane; e < BN * U; e += 32) {
                    const int r = e / U;
                    uint4 *at = (uint4 *)(vt + bf16_off<D>(r, (e % U) * 8));
                    if (r >= valid) {
                        *at = make_uint4(0, 0, 0, 0);
                        continue;
                    }
                    const uint4 v = *at;
                    uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    bool any = false;
#pragma unroll
                    for (int k = 0; k < 4; ++k) any = any || (w[k] & 0x7f80u) == 0x7f80u || (w[k] & 0x7f800000u) == 0x7f800000u;
                    if (!any) continue;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if ((w[k] & 0x7f80u) == 0x7f80u) w[k] &= 0xffff0000u;
                        if ((w[k] & 0x7f800000u) == 0x7f800000u) w[k] &= 0xffffu;
                        if (r >> 5 == k) bad[k] |= 1u << (r & 31);
                    }
                    *at = make_uint4(w[0], w[1], w[2], w[3]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) bad[k] = __reduce_or_sync(0xffffffffu, bad[k]);
                if ((bad[0] | bad[1] | bad[2] | bad[3]) && lane == 0 && sh.n_bad[ub] < kBadTiles) {
                    const int i = sh.n_bad[ub];
                    for (int k = 0; k < 4; ++k) sh.bad[ub][i][k] = bad[k];
                    sh.bad_key[ub][i] = j * BN;
                    sh.n_bad[ub] = i + 1;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_addr(&sh.v_clean[st]));
                    mbar_arrive(smem_addr(&sh.v_free[st]));
                }
            }
        } else if (warp >= C::MMA_WARP) {
            // ---- products ----
            const int slot = warp - C::MMA_WARP;
            const bool live = rows_here > slot * kTileRows && u.rq.seq >= 0;
            if (lane == 0) {
                const uint32_t id_s = idesc_f16(!Q8, false, BN), id_o = idesc_f16(!Q8, true, D);
                const uint32_t q_addr = smem_addr(smem) + slot * C::Q_BYTES, k_addr = smem_addr(smem + C::OFF_K), v_addr = smem_addr(smem + C::OFF_V);
                const uint32_t cols = tmem + (uint32_t)(slot * C::SLOT_COLS);
                auto issue_s = [&](int i) {  // tile i of the unit
                    const int at = it + i, st = at % NS;
                    if (!mbar_wait(smem_addr(&sh.full_k[st]), (at / NS) & 1, abort, kWait)) return false;
                    if (!live) {
                        mbar_arrive(smem_addr(&sh.s_full[slot][st]));
                        return true;
                    }
                    tc_fence_after();
                    const uint32_t s_at = cols + (uint32_t)(C::S_COL + ((live_it[0] + i) % NSB) * BN);
                    const uint64_t qa = sdesc(q_addr, 16, C::SBO, C::LAYOUT), kb = sdesc(k_addr + st * C::KV_BYTES, 16, C::SBO, C::LAYOUT);
#pragma unroll
                    for (int s4 = 0; s4 < D / 64; ++s4) {
                        uint64_t av[4], bv[4];
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            av[s] = qa + ((uint32_t)(s4 * 1024 + s * 32) >> 4);
                            bv[s] = kb + ((uint32_t)(s4 * 1024 + s * 32) >> 4);
                        }
                        mma_ss_x4<false>(s_at, av, bv, id_s, s4 > 0 ? 1u : 0u);
                    }
                    mma_commit(smem_addr(&sh.s_full[slot][st]));
                    return true;
                };
                auto issue_pv = [&](int i) {
                    const int at = it + i, st = at % NS;
                    if (live && !mbar_wait(smem_addr(&sh.p_full[slot][(live_it[0] + i) % NSB]), ((live_it[0] + i) / NSB) & 1, abort, kWait)) return false;
                    if (!mbar_wait(smem_addr(&sh.full_v[st]), (at / NS) & 1, abort, kWait)) return false;
                    if (!Q8 && !unit_sees(t0 + i)) {
                        if (!mbar_wait(smem_addr(&sh.v_clean[st]), (clean_phase >> st) & 1u, abort, kWait)) return false;
                        clean_phase ^= 1u << st;
                    }
                    if (!live) {
                        mbar_arrive(smem_addr(&sh.v_free[st]));
                        return true;
                    }
                    tc_fence_after();
                    const uint32_t p_at = cols + (uint32_t)(C::S_COL + ((live_it[0] + i) % NSB) * BN);
                    const uint64_t vb = sdesc(v_addr + st * C::KV_BYTES, 1024, C::SBO, C::LAYOUT);
#pragma unroll
                    for (int s4 = 0; s4 < BN / 64; ++s4) {
                        uint32_t av[4];
                        uint64_t bv[4];
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            const int k = 4 * s4 + s;  // 16 keys; P of a warp's keys starts where their S did
                            av[s] = p_at + (uint32_t)(16 * k / KPW * KPW + 16 * k % KPW / 2);
                            bv[s] = vb + ((uint32_t)(k * 2 * C::SBO) >> 4);
                        }
                        mma_ts_x4<false>(cols + C::O_COL, av, bv, id_o, i > 0 || s4 > 0 ? 1u : 0u);
                    }
                    mma_commit(smem_addr(&sh.v_free[st]));
                    return true;
                };
                // S(j + NSB) goes over P(j), whose product is issued before it: the tensor pipe runs them in order
                if (live) ok = ok && mbar_wait(smem_addr(&sh.q_ready[slot]), live_units & 1, abort, kWait);
                for (int i = 0; ok && i < min(NSB, n); ++i) ok = issue_s(i);
                for (int i = 0; ok && i < n; ++i) {
                    ok = issue_pv(i);
                    if (ok && i + NSB < n) ok = issue_s(i + NSB);
                }
                if (live) mma_commit(smem_addr(&sh.o_done[slot]));
                if (!ok) *abort = 1;
            }
            it += n;
            if (live) {
                live_it[0] += n;
                ++live_units;
            }
        } else {
            // ---- softmax: thread = row and half of the tile's keys ----
            const int slot = warp >> 3, quarter = warp & 3, half = (warp >> 2) & 1, r = quarter * 32 + lane;
            const int row = u.row0 + slot * kTileRows + r, t = row_token(a, row), id = 1 + slot * 4 + quarter;
            const bool slot_live = rows_here > slot * kTileRows && u.rq.seq >= 0;
            const bool on = row < u.rows_all;
            const int64_t src_row = (int64_t)a.src_row[u.b] + t;
            const int head = u.g * a.group + row - t * a.group;
            if (!slot_live) {
                for (int i = 0; i < n; ++i, ++it) ok = ok && warp_wait(smem_addr(&sh.s_full[slot][it % NS]), (it / NS) & 1, abort);
                if (!ok) *abort = 1;
                if (u.rq.seq < 0 && on && t0 == 0) {  // a refused request's rows are 0
                    for (int c = half * D / 2; c < (half + 1) * D / 2; c += 8)
                        *(uint4 *)(a.out + (src_row * a.q_heads + head) * D + c) = make_uint4(0, 0, 0, 0);
                }
                ++unit_no;
                continue;
            }
            const uint32_t lane_base = ((uint32_t)(quarter * 32) << 16) + (uint32_t)(slot * C::SLOT_COLS);
            const bool live = __any_sync(0xffffffffu, on);  // (a pair's two warps have the same rows)
            float *const mine = s_x + (slot * 2 + half) * kTileRows, *const other = s_x + (slot * 2 + (half ^ 1)) * kTileRows;
            {
                // query rows: this warp those of its lane quarter's half
                constexpr int U = D / 8;
                uint8_t *sq = smem + slot * C::Q_BYTES;
                const long long at = (long long)src_row * a.q_stride + (long long)head * D;
                const uint32_t have = __ballot_sync(0xffffffffu, on);
#pragma unroll 8
                for (int i = lane; i < 16 * U; i += 32) {
                    const int rr = half * 16 + i / U, uu = i % U;
                    const long long from = __shfl_sync(0xffffffffu, at, rr);
                    const bool has = (have >> rr) & 1u;
                    uint8_t *to = sq + bf16_off<D>(quarter * 32 + rr, 8 * uu);
                    if constexpr (!Q8) {
                        cp_async_16_or_zero(smem_addr(to), has ? a.q + from + 8 * uu : a.q, has);
                    } else {
                        const uint4 v = has ? *(const uint4 *)(a.q + from + 8 * uu) : make_uint4(0, 0, 0, 0);
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                        uint32_t o[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float lo = __uint_as_float(w[k] << 16), hi = __uint_as_float(w[k] & 0xffff0000u);
                            fits = fits && fabsf(lo) <= 65504.0f && fabsf(hi) <= 65504.0f;
                            const __half2 h = __floats2half2_rn(lo, hi);
                            o[k] = *(const uint32_t *)&h;
                        }
                        *(uint4 *)to = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
                if (!Q8) cp_async_wait_all();
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&sh.q_ready[slot]));
            }
            float m = -INFINITY;
            uint64_t l0 = 0, l1 = 0;  // the row's sum over this warp's keys
            const int p = u.rq.pos0 + t;
            for (int i = 0; i < n; ++i, ++it) {
                const int st = it % NS, j = t0 + i, sb = (live_it[0] + i) % NSB;
                ok = ok && warp_wait(smem_addr(&sh.s_full[slot][st]), (it / NS) & 1, abort);
                if (!ok) *abort = 1;
                tc_fence_after();
                const uint32_t s_col = tmem + lane_base + (uint32_t)(C::S_COL + sb * BN + half * KPW);
                if (live) {
                    uint32_t s[KPW];
                    if constexpr (KPW == 64) tmem_load32x2(s_col, s_col + 32, *(uint32_t(*)[32])s, *(uint32_t(*)[32])(s + 32));
                    else tmem_load32(s_col, *(uint32_t(*)[32])s);
                    if (!unit_sees(j)) {
#pragma unroll
                        for (int c = 0; c < KPW; c += 32) {
                            const uint32_t bits = on ? seen_bits(a, sp, p, j * BN + half * KPW + c) : 0u;
#pragma unroll
                            for (int k = 0; k < 32; ++k)
                                if (!((bits >> k) & 1u)) s[c + k] = 0xff800000u;
                        }
                    }
                    float top = -INFINITY, top1 = -INFINITY;
#pragma unroll
                    for (int k = 0; k < KPW; k += 4) {
                        top = max3(top, __uint_as_float(s[k]), __uint_as_float(s[k + 1]));
                        top1 = max3(top1, __uint_as_float(s[k + 2]), __uint_as_float(s[k + 3]));
                    }
                    top = fmaxf(top, top1);
                    const float mt = top == -INFINITY ? -INFINITY : top * a.scale_log2;
                    // m moves when a score of either warp's keys is more than 2^8 above it
                    if (pair_any(id, mt > m + 8.0f)) {
                        mine[r] = mt;
                        pair_sync(id);
                        const float mn = fmaxf(mt, other[r]);
                        const bool up = mn > m + 8.0f;
                        const float f = up ? ex2(m - mn) : 1.0f;  // (0 for the first)
                        if (up) m = mn;
                        l0 = fma_pair(l0, pair_of(f, f), 0);
                        l1 = fma_pair(l1, pair_of(f, f), 0);
                        if (i > 0 && __any_sync(0xffffffffu, up)) {
                            // O of the tiles before is complete: with one S tile because S came after it, with two it is waited for
                            if (NSB > 1) {
                                ok = ok && warp_wait(smem_addr(&sh.v_free[(it - 1) % NS]), ((it - 1) / NS) & 1, abort);
                                tc_fence_after();
                            }
#pragma unroll 1
                            for (int c0 = half * D / 2; c0 < (half + 1) * D / 2; c0 += 32) {
                                uint32_t o[32];
                                tmem_load32(tmem + lane_base + C::O_COL + c0, o);
#pragma unroll
                                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                                tmem_st32(tmem + lane_base + C::O_COL + c0, o);
                            }
                        }
                    }
                    const float neg = m == -INFINITY ? 0.0f : -m;
                    const uint64_t scale2 = pair_of(a.scale_log2, a.scale_log2), neg2 = pair_of(neg, neg);
#pragma unroll
                    for (int c = 0; c < KPW; c += 32) {
                        uint32_t w[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float2 v = of_pair(fma_pair(pair_of(__uint_as_float(s[c + 2 * k]), __uint_as_float(s[c + 2 * k + 1])), scale2, neg2));
                            v = make_float2(ex2(v.x), ex2(v.y));
                            uint64_t add;
                            if constexpr (Q8) {
                                const __half2 h = __floats2half2_rn(v.x, v.y);
                                w[k] = *(const uint32_t *)&h;
                                add = pair_of(v.x, v.y);
                            } else {
                                w[k] = pack_bf16(v.x, v.y);
                                add = pair_of(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
                            }
                            if (k & 1) l1 = add_pair(l1, add);
                            else l0 = add_pair(l0, add);
                        }
                        tmem_st16(s_col + c / 2, w);
                    }
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&sh.p_full[slot][sb]));
            }
            live_it[0] += n;
            ok = ok && warp_wait(smem_addr(&sh.o_done[slot]), live_units & 1, abort);
            ++live_units;
            if (!ok) *abort = 1;
            tc_fence_after();
            const float2 la = of_pair(l0), lb = of_pair(l1);
            const float part_l = (la.x + la.y) + (lb.x + lb.y);
            if (live) {
                pair_sync(id);  // (maxima have been read)
                mine[r] = part_l;
                pair_sync(id);
            }
            if (ok && live) {
                const float l = part_l + other[r];
                const bool whole = t0 == 0 && t1 == n_tiles;
                const long long part = (2ll * blockIdx.x + (t0 == 0 ? 1 : 0)) * ROWS + slot * kTileRows + r;
                if (!whole && half == 0 && on) a.ws_ml[part] = make_float4(m, l, 0.0f, 0.0f);
                const float f = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
                const int ub = unit_no % kBadUnits, n_bad = Q8 ? 0 : *(volatile int *)&sh.n_bad[ub];
                uint16_t *const out = a.out + (src_row * a.q_heads + head) * D;
#pragma unroll 1
                for (int c0 = half * D / 2; c0 < (half + 1) * D / 2; c0 += 32) {
                    uint32_t o[32];
                    __syncwarp();
                    tmem_load32(tmem + lane_base + C::O_COL + c0, o);
                    // rare: values that are not finite, for the rows that see them
#pragma unroll 1
                    for (int i = 0; i < n_bad; ++i)
#pragma unroll 1
                        for (int k = 0; k < BN; ++k) {
                            if (!((sh.bad[ub][i][k >> 5] >> (k & 31)) & 1u)) continue;
                            const int key = sh.bad_key[ub][i] + k, slot_k = sp.slot(key);
                            if (!on || !(seen_bits(a, sp, p, key) & 1u)) continue;
                            const int e = slot_k / a.pool.block_tokens, blk = lookup_block(a.pool, u.rq.seq, e);
                            if (blk < 0) continue;
                            const uint8_t *tile = a.pool.prefix + prefix_tile_index(a.pool, a.layer, blk, 1, u.g) * a.pool.tile_bytes;
#pragma unroll
                            for (int c = 0; c < 32; ++c) {
                                const float y = bf16_bits_to_f32(*(const uint16_t *)(tile + bf16_off<D>(slot_k - e * a.pool.block_tokens, c0 + c)));
                                if (!isfinite(y)) o[c] = __float_as_uint(__uint_as_float(o[c]) + y);
                            }
                        }
                    // a row without a key has nothing (not 0 * what the columns hold)
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = l != 0.0f ? __float_as_uint(__uint_as_float(o[k]) * f) : 0u;
                    if (on && !whole) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4) *(uint4 *)(a.ws_o + part * D + c0 + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                    } else if (on) {
#pragma unroll
                        for (int k = 0; k < 32; k += 8) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] = pack_bf16(__uint_as_float(o[k + 2 * e]), __uint_as_float(o[k + 2 * e + 1]));
                            *(uint4 *)(out + c0 + k) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
                __syncwarp();
            }
            if (a.split && threadIdx.x == 0 && t0 == 0) {  // the CTAs of this unit: tile x is CTA ((x + 1) G - 1) / T's
                const unsigned long long end = (unsigned long long)base + (uint32_t)(u.g + 1) * (uint32_t)n_tiles;
                a.parts[(long long)flat * hk + u.g] = make_int2(blockIdx.x, (int)((end * rg.ctas - 1) / rg.total));
            }
            tc_fence_before();
        }
        ++unit_no;
    }
    if (!ok && lane == 0) report_error(a.pool.status, DEV_ERR_TIMEOUT, blockIdx.x, warp, 15);
    if (!__all_sync(0xffffffffu, fits) && lane == 0) report_error(a.pool.status, DEV_ERR_F16_RANGE, blockIdx.x, warp, 15);
    if (warp >= C::FEED_WARP && warp < (Q8 ? C::CONV_WARP : C::SCRUB_WARP) && !ok && lane == 0) {
        // leave no copy writing this CTA's shared memory
        for (int i = 0; i < (Q8 ? C::NR : NS); ++i) {
            const uint32_t bar = smem_addr(Q8 ? &sh.raw_full[i] : warp == C::FEED_WARP ? &sh.full_k[i] : &sh.full_v[i]);
            mbar_wait_drain(bar, 0, kWait / 64);
            mbar_wait_drain(bar, 1, kWait / 64);
        }
    }
    if (warp >= C::MMA_WARP && warp < C::FEED_WARP && lane == 0) {  // nor a product using its tensor memory
        mma_commit(smem_addr(&sh.drained[warp - C::MMA_WARP]));
        mbar_wait_drain(smem_addr(&sh.drained[warp - C::MMA_WARP]), 0, kWait);
    }
    __syncthreads();
    if (warp == C::MMA_WARP) tmem_dealloc(tmem, C::COLS);
}

template <int D, bool Q8>
int launch_form(const WindowArgs &a, int grid, cudaStream_t s) {
    using C = WCfg<D, Q8>;
    static std::atomic<uint64_t> done{0};
    if (const int rc = allow_smem(window_tile_kernel<D, Q8>, C::SMEM, done)) return rc;
    return launch_after(window_tile_kernel<D, Q8>, grid, C::THREADS, C::SMEM, s, a);
}

}  // namespace

int window_tile_rows(int head_dim) { return (head_dim > 128 ? 1 : 2) * kTileRows; }
int window_tile_keys(int head_dim) { return head_dim > 128 ? 64 : 128; }

int launch_window_tile(const WindowArgs &a, int grid, cudaStream_t s) {
    const bool q8 = a.pool.dtype == EKV_DTYPE_Q8_0;
    switch (a.pool.head_dim) {
        case 64: return q8 ? launch_form<64, true>(a, grid, s) : launch_form<64, false>(a, grid, s);
        case 128: return q8 ? launch_form<128, true>(a, grid, s) : launch_form<128, false>(a, grid, s);
        case 256: return q8 ? launch_form<256, true>(a, grid, s) : launch_form<256, false>(a, grid, s);
        default: return EKV_ERR_UNSUPPORTED;
    }
}

}  // namespace ekv
