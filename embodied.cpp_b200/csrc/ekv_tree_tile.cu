// ekv_tree_tile.cu -- draft-tree attention for many query rows per KV head, on tcgen05.
//
// The same sums as ekv_tree.cu. With many rows per cached key the products bound the call, not the bytes, so row
// tiles of 128 take the 5th-generation tensor cores (from 17 rows on: tree_tile_rows()): S = Q K^T with both operands in shared memory and S
// in tensor memory, P = exp(S - m) as bf16 over S's own columns, O += P V with P read from tensor memory.
// Four warps are the softmax of a 128-row tile (a thread is a row) and one more issues its products; one feeds K
// and V through the copy engine (pool tiles are canonical operands as they are stored).
// A row tile has two S tiles of 64 keys, so that S(j + 1) is computed under the exponentials of S(j); and
// exponentials and products take about as long (64 keys of 128 rows at head_dim 128: 512 cycles of the one, 640 of
// the other), so two row tiles share an SM and take turns on both pipes:
//   RT = 2 (head_dim 64 or 128, more than 128 rows): one CTA holds two row tiles of a KV head, which read each
//     K/V tile once between them; 256 tensor-memory columns each.
//   RT = 1 (up to 128 rows): two CTAs per SM of one row tile each; at head_dim 256 one CTA, by its size.
// With one S tile of 128 keys per row tile instead, the chain S, maximum, exponentials, P V left the tensor pipe
// idle half of the time: 4300 cycles per 128 keys of two row tiles. With one issuing warp for both row tiles its
// barrier waits, about 220 idle cycles each, took half: 5080 cycles.
// Bound and figures: 8 requests of 8192 keys, 8 KV heads of 128 columns, 256 rows each (62 GFLOP, 258 MB) take 72 us and
// 11 of the join, 750 TFLOP/s. 64 keys of two row tiles take 1980 cycles of the products' 1280: no pipe is full (tensor
// memory and cores 55%, exponentials 41%, issue 45%), the softmax warps' chain of waits and tensor-memory reads is what
// is left. Loading S of the next tile under the exponentials, with P in columns of its own, made it longer (2300 cycles);
// exponentials and sums in a fixed order, or row tiles half a tile apart, changed nothing.
#include "ekv_decode.cuh"

namespace ekv {
namespace {

using namespace decode;
using namespace sm100;

// Q8: pages of 8-bit blocks. A value of one, int8 times an f16 scale, has up to 19 significant bits, so K and V are two
// bf16 tiles each, the value rounded and what that left (2^-17 of it at most is lost), and each product is two: the
// scores stay as exact as the rows kernel's. Eight warps make them from the blocks that the feeder brought, K before V,
// so that S of the next tile waits neither for V nor behind the product before it (one barrier for both: 204 us instead
// of 158 for 32 rows of 16 requests of 4096 keys, 8 KV heads of 128 columns), and Q lies in tensor memory (152 us). 64 keys
// take 4200 cycles of an SM: 2600 of conversion, and products at half their rate beside its shared-memory writes.
template <int D, int RT, bool Q8>
struct TCfg {
    static constexpr int BN = kTile, NSB = 2;                   // keys per tile; S tiles per row tile
    static constexpr int NS = RT == 2 || D == 64 ? 4 : 2;          // K and V stages
    static constexpr int CTAS = D > 128 || RT == 2 || Q8 ? 1 : 2;  // per SM
    static constexpr uint32_t SBO = 16 * D;        // bytes between 8-row groups; chunks of 64 columns are 1024 apart
    static constexpr uint32_t LAYOUT = 2;          // 128-byte swizzle
    static constexpr int PARTS = Q8 ? 2 : 1;       // of K and V
    static constexpr int PART_BYTES = BN * D * 2, KV_BYTES = PARTS * PART_BYTES;
    static constexpr int NR = Q8 ? 3 : 1;          // stages of blocks as they are stored, K then V (Q8)
    static constexpr int RAW_KV = (TileCfg<D, true>::KV_BYTES + 127) / 128 * 128;
    static constexpr int Q_BYTES = kTreeTileRows * D * 2;
    static constexpr int SLOT_COLS = 256;          // tensor-memory columns from row tile to row tile
    static constexpr int S_COL = 0, O_COL = BN * NSB, Q_COL = O_COL + D;
    static constexpr int COLS = D > 128 || (Q8 && D == 128) ? 512 : SLOT_COLS * RT;
    static constexpr int OFF_K = RT * Q_BYTES, OFF_V = OFF_K + NS * KV_BYTES;
    static constexpr int OFF_RAW = OFF_V + NS * KV_BYTES, OFF_SH = OFF_RAW + (Q8 ? (NR * 2 * RAW_KV + 1023) / 1024 * 1024 : 0);
    static constexpr int SMEM = OFF_SH + 2048 + 1024;
    static constexpr int ROW_WARPS = 4 * RT, MMA_WARP = ROW_WARPS, FEED_WARP = ROW_WARPS + RT;
    static constexpr int CONV_WARP = FEED_WARP + 1, CONV_WARPS = Q8 ? 8 : 0, THREADS = (CONV_WARP + CONV_WARPS) * 32;
    static_assert(O_COL + D <= (D > 128 ? 512 : SLOT_COLS), "tensor memory");
    static_assert(D % 64 == 0 && (RT == 1 || D <= 128), "whole swizzle chunks; two outputs fit");
    static_assert(!Q8 || (RT == 1 && D <= 128), "shared memory");
};

// Phases: full, s_full, v_done and v_clean go by the tile's stage (tile / NS), p_full by its S tile (tile / NSB),
// q_ready by the CTA's unit. The two row tiles run at most NS tiles apart, as a stage is refilled after both.
struct TShared {
    uint64_t full[4];       // K and V of the stage have landed (Q8: K)
    uint64_t full_v[4];     // Q8: V
    uint64_t raw_full[3], raw_empty[3];  // blocks have landed; are converted
    uint64_t s_full[2][4];  // [row tile][stage] S done
    uint64_t v_done[2][4];  // [row tile][stage] P V done
    uint64_t p_full[2][2];  // [row tile][S tile] P written
    uint64_t q_ready[2];    // [row tile] query rows in shared memory
    uint64_t v_clean[4];    // the first row tile's warps have made rows without a key zero and taken what is not
                            // finite out of the drafts
    uint64_t drained[2];
    unsigned long long bad[8];  // [unit % 8] drafted keys of the unit whose values are not all finite
    uint32_t tmem;
    int abort;
    RangeScratch range;
    int table[kTableWindow];
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Visible columns [0, 32) of a 32-column chunk that starts at key c0 of the tile: `word` has a bit per key.
__device__ __forceinline__ uint32_t chunk_bits(unsigned long long word, int c0, int valid) {
    const uint32_t w = c0 >= 64 ? 0xffffffffu : (uint32_t)(word >> c0);
    const int n = valid - c0;
    return n >= 32 ? w : n <= 0 ? 0u : w & ((1u << n) - 1u);
}

// A Q8_0 block's rows as two bf16 tiles: 16 columns at a time, four of them and two rows in every eight lanes, which
// then write to eight different 16-byte columns of the swizzled rows.
template <int D, int THREADS>
__device__ __forceinline__ void convert_tile(const uint8_t *raw, uint8_t *dst, int part_bytes, int valid, int thread) {
    constexpr int U = D / 16;
#pragma unroll 2
    for (int e = thread; e < kTile * U; e += THREADS) {
        const int rest = e >> 3, u = (rest % (U / 4)) * 4 + (e & 3), row = rest / (U / 4) * 2 + ((e >> 2) & 1);
        uint32_t hi[8] = {}, lo[8] = {};
        if (row < valid) {
            const uint4 v = *(const uint4 *)(raw + q8_qs_off(row, 16 * u, D));
            const float d = __half2float(*(const __half *)(raw + TileCfg<D, true>::SCALES + (row * (D / 32) + (u >> 1)) * 2));
            const bool finite = fabsf(d) < INFINITY;
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t q[2];
                int8x4_to_bf16(w[i], q[0], q[1]);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint64_t x = fma_pair(pair_of(__uint_as_float(q[k] << 16), __uint_as_float(q[k] & 0xffff0000u)), pair_of(d, d), 0);
                    const uint32_t h = pack_bf16(of_pair(x).x, of_pair(x).y);
                    const float2 r = of_pair(fma_pair(pair_of(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)), pair_of(-1.0f, -1.0f), x));
                    hi[2 * i + k] = h;
                    lo[2 * i + k] = finite ? pack_bf16(r.x, r.y) : 0u;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t off = bf16_off<D>(row, 16 * u + 8 * k);
            *(uint4 *)(dst + off) = make_uint4(hi[4 * k], hi[4 * k + 1], hi[4 * k + 2], hi[4 * k + 3]);
            *(uint4 *)(dst + part_bytes + off) = make_uint4(lo[4 * k], lo[4 * k + 1], lo[4 * k + 2], lo[4 * k + 3]);
        }
    }
}

// FINE (f32 outputs): P as two bf16 parts, the second over the 32 columns of S that the first leaves (8 requests of 8192 keys,
// 8 KV heads of 128 columns, 256 rows each 86.7 -> 90.1 us; 16 of 4096 8-bit keys 295 -> 311).
template <int D, int RT, bool Q8, bool CAP, bool FINE>
__global__ void __launch_bounds__(TCfg<D, RT, Q8>::THREADS, TCfg<D, RT, Q8>::CTAS) tree_tile_kernel(const TreeArgs a) {
    using C = TCfg<D, RT, Q8>;
    constexpr int BN = C::BN, NS = C::NS, NSB = C::NSB, ROWS = RT * kTreeTileRows;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    TShared &sh = *(TShared *)(smem + C::OFF_SH);
    static_assert(sizeof(TShared) <= 2048, "barrier block");
    volatile int *abort = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hk = a.pool.kv_heads, units_per_req = hk * a.row_tiles;
    const int rows_all = a.n_draft * a.group;

    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(smem_addr(&sh.full[i]), Q8 ? C::CONV_WARPS : 2);
            if (Q8) mbar_init(smem_addr(&sh.full_v[i]), C::CONV_WARPS);
            mbar_init(smem_addr(&sh.v_clean[i]), 4);
            for (int k = 0; k < RT; ++k) {
                mbar_init(smem_addr(&sh.s_full[k][i]), 1);
                mbar_init(smem_addr(&sh.v_done[k][i]), 1);
            }
        }
        for (int k = 0; k < RT; ++k) {
            for (int i = 0; i < NSB; ++i) mbar_init(smem_addr(&sh.p_full[k][i]), 4);
            mbar_init(smem_addr(&sh.q_ready[k]), 4);
            mbar_init(smem_addr(&sh.drained[k]), 1);
        }
        for (int i = 0; Q8 && i < C::NR; ++i) {
            mbar_init(smem_addr(&sh.raw_full[i]), 2);
            mbar_init(smem_addr(&sh.raw_empty[i]), C::CONV_WARPS);
        }
        sh.abort = 0;
        mbar_init_fence();
    }
    auto unit_tiles = [](const Req &r) { return max(1, (r.n_prefix + BN - 1) / BN + (r.n_nodes > 0 ? 1 : 0)); };
    grid_wait();
    // Tensor memory is taken between the two launch points: before the wait this CTA could hold columns that a CTA of the
    // kernel it waits for still has to get, and after the signal a CTA of the next kernel could hold this one's.
    if (warp == C::MMA_WARP) tmem_alloc(smem_addr(&sh.tmem), C::COLS);
    tc_fence_before();
    Range rg;
    if (a.split) {
        rg = find_range<C::THREADS>(a.n_batch, units_per_req, sh.range,
                                      [&](int b) { return load_req(a, b, blockIdx.x == 0); }, unit_tiles);
    } else {
        __syncthreads();
        rg.b = blockIdx.x / units_per_req;
        rg.req = load_req(a, rg.b, threadIdx.x == 0);
        const int n = unit_tiles(rg.req);
        rg.base = 0;
        rg.lo = (blockIdx.x - rg.b * units_per_req) * (uint32_t)n;
        rg.hi = rg.lo + n;
        rg.total = 0;
        rg.ctas = 0;
    }
    tc_fence_after();
    const uint32_t tmem = sh.tmem;  // (there is a barrier in either branch)
    grid_launch_next();

    int it = 0, unit_no = 0;  // tiles and units of this CTA so far
    int raw_it = 0;           // tiles of blocks (the feeder's and the converters')
    bool ok = true;
    TableWindow tw;  // (the feeder's)
    tw.reset(sh.table);
    int b = rg.b;
    uint32_t base = rg.base;
    Req rq = rg.req;
    int rq_of = b;  // the request that rq describes
    for (uint32_t x = rg.lo; x < rg.hi && b < a.n_batch;) {
        if (b != rq_of) rq = load_req(a, b, false), rq_of = b;
        const int n_tiles = unit_tiles(rq);
        const uint32_t span = (uint32_t)n_tiles * units_per_req;
        if (x >= base + span) {
            base += span;
            ++b;
            continue;
        }
        const int u = (int)((x - base) / (uint32_t)n_tiles);
        const int t0 = (int)(x - base) - u * n_tiles;
        const int t1 = min(n_tiles, t0 + (int)(rg.hi - x));
        const int n = t1 - t0;
        const int g = u / a.row_tiles, row0 = (u - g * a.row_tiles) * ROWS;
        const int p_tiles = (rq.n_prefix + BN - 1) / BN;
        const long long kv_row = ((long long)b * a.n_draft * hk + g) * D;
        auto tile_full = [&](int j) { return (j + 1) * BN <= rq.n_prefix; };

        if (warp == C::FEED_WARP) {
            // ---- feeder ----
            Piece next = find_piece<D, Q8>(a, rq, g, t0 * BN, tw, lane);
            if (a.split && lane == 0 && t0 == 0) {  // the CTAs of this unit: tile x is CTA ((x + 1) G - 1) / T's
                const unsigned long long end = base + (uint32_t)(u + 1) * n_tiles;
                a.parts[b * units_per_req + u] = make_int2(blockIdx.x, (int)((end * rg.ctas - 1) / rg.total));
            }
            for (int j = t0; j < t1; ++j, ++it) {
                const int st = it % NS, par = (it / NS) & 1;
                const Piece pc = next;
                if (j + 1 < min(t1, p_tiles)) next = find_piece<D, Q8>(a, rq, g, (j + 1) * BN, tw, lane);
                if constexpr (Q8) {
                    if (j >= p_tiles) continue;  // (drafted rows are the converters')
                    const int rs = raw_it % C::NR;
                    if (raw_it >= C::NR) ok = ok && warp_wait(smem_addr(&sh.raw_empty[rs]), (raw_it / C::NR - 1) & 1, abort);
                    if (!ok) {
                        *abort = 1;
                        continue;
                    }
                    const uint32_t raw = smem_addr(smem + C::OFF_RAW + rs * 2 * C::RAW_KV), bar = smem_addr(&sh.raw_full[rs]);
                    issue_piece<D, true, true>(a, pc, raw, raw + C::RAW_KV, bar, bar, lane);
                    ++raw_it;
                    continue;
                }
                const uint32_t sk = smem_addr(smem + C::OFF_K + st * C::KV_BYTES);
                const uint32_t sv = smem_addr(smem + C::OFF_V + st * C::KV_BYTES);
                const uint32_t bar = smem_addr(&sh.full[st]);
                if (NS < 4 && pc.src && j < p_tiles)  // the stage may be taken for a while: start the way from memory
                    bulk_prefetch_l2(pc.src + pc.rib * D * 2, (uint32_t)(pc.n * D * 2));
                if (it >= NS) {
#pragma unroll
                    for (int k = 0; k < RT; ++k) ok = ok && warp_wait(smem_addr(&sh.v_done[k][st]), par ^ 1, abort);
                }
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                if (j < p_tiles) {
                    issue_piece<D, false, true>(a, pc, sk, sv, bar, bar, lane);
                    continue;
                }
                // drafted rows, from the caller's buffers: a lane keeps its 16-byte unit of the rows
                const int nd = rq.n_nodes;
                constexpr int U = D / 8, AT_ONCE = 32 / U > 0 ? 32 / U : 1;
#pragma unroll
                for (int u0 = 0; u0 < U; u0 += 32) {
                    const int uu = u0 + lane % (U < 32 ? U : 32), r0 = U < 32 ? lane / U : 0;
                    const long long src = kv_row + (long long)r0 * hk * D + 8 * uu;
                    const uint16_t *kp = a.k_draft + src, *vp = a.v_draft + src;
                    const long long step = (long long)AT_ONCE * hk * D;
#pragma unroll 8
                    for (int r = r0; r < nd; r += AT_ONCE) {
                        const uint32_t off = bf16_off<D>(r, 8 * uu);
                        cp_async_16(sk + off, kp);
                        cp_async_16(sv + off, vp);
                        kp += step;
                        vp += step;
                    }
                }
                cp_async_wait_all();
                fence_proxy_async();  // read by the tensor core
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar);
                    mbar_arrive(bar);
                }
            }
        } else if (Q8 && warp >= C::CONV_WARP) {
            // ---- converters: K of a tile once S of the tile before it in its stage is done, V once that tile's P V is ----
            const int thread = threadIdx.x - C::CONV_WARP * 32;
            for (int j = t0; j < t1; ++j, ++it) {
                const int st = it % NS, rs = raw_it % C::NR;
                const bool draft = j >= p_tiles;
                const int valid = draft ? rq.n_nodes : min(BN, rq.n_prefix - j * BN);
                const uint8_t *raw = smem + C::OFF_RAW + rs * 2 * C::RAW_KV;
                if (!draft) ok = ok && warp_wait(smem_addr(&sh.raw_full[rs]), (raw_it / C::NR) & 1, abort);
#pragma unroll 1
                for (int v = 0; v < 2; ++v) {
                    const uint32_t before = smem_addr(v ? &sh.v_done[0][st] : &sh.s_full[0][st]);
                    if (it >= NS) ok = ok && warp_wait(before, (it / NS - 1) & 1, abort);
                    if (!ok) break;
                    uint8_t *dst = smem + (v ? C::OFF_V : C::OFF_K) + st * C::KV_BYTES;
                    if (!draft) {
                        convert_tile<D, C::CONV_WARPS * 32>(raw + v * C::RAW_KV, dst, C::PART_BYTES, valid, thread);
                    } else {  // bf16 already: one part; rows past the last are zero
                        constexpr int U = D / 8;
                        const uint16_t *rows = (v ? a.v_draft : a.k_draft) + kv_row;
                        for (int e = thread; e < BN * U; e += C::CONV_WARPS * 32) {
                            const int r = e / U, u = e % U;
                            *(uint4 *)(dst + bf16_off<D>(r, 8 * u)) =
                                r < valid ? *(const uint4 *)(rows + (long long)r * hk * D + 8 * u) : make_uint4(0, 0, 0, 0);
                        }
                    }
                    fence_proxy_async();  // read by the tensor core
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_addr(v ? &sh.full_v[st] : &sh.full[st]));
                }
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                if (!draft) {
                    if (lane == 0) mbar_arrive(smem_addr(&sh.raw_empty[rs]));
                    ++raw_it;
                }
            }
        } else if (warp >= C::MMA_WARP) {
            // ---- products ----
            const int slot = warp - C::MMA_WARP;
            if (lane == 0) {
                const uint32_t id_s = idesc_f16(true, false, BN), id_o = idesc_f16(true, true, D);
                const uint32_t q_addr = smem_addr(smem), k_addr = smem_addr(smem + C::OFF_K), v_addr = smem_addr(smem + C::OFF_V);
                auto s_at = [&](int i) { return tmem + (uint32_t)(slot * C::SLOT_COLS + C::S_COL + (i % NSB) * BN); };
                auto parts_of = [&](int i) { return t0 + i - it >= p_tiles ? 1 : C::PARTS; };  // (drafts have one)
                auto issue_s = [&](int i) {
                    const int st = i % NS;
                    if (!mbar_wait(smem_addr(&sh.full[st]), (i / NS) & 1, abort, kWait)) return false;
                    tc_fence_after();
                    const uint64_t qa = sdesc(q_addr + slot * C::Q_BYTES, 16, C::SBO, C::LAYOUT);
                    const uint64_t kb = sdesc(k_addr + st * C::KV_BYTES, 16, C::SBO, C::LAYOUT);
#pragma unroll
                    for (int part = 0; part < C::PARTS; ++part) {
                        if (part >= parts_of(i)) break;
#pragma unroll
                        for (int s4 = 0; s4 < D / 64; ++s4) {  // four 16-column steps of a 64-column chunk
                            uint64_t av[4], bv[4];
                            uint32_t qt[4];
#pragma unroll
                            for (int s = 0; s < 4; ++s) {
                                av[s] = qa + ((uint32_t)(s4 * 1024 + s * 32) >> 4);
                                qt[s] = tmem + (uint32_t)(C::Q_COL + (4 * s4 + s) * 8);
                                bv[s] = kb + ((uint32_t)(part * C::PART_BYTES + s4 * 1024 + s * 32) >> 4);
                            }
                            const uint32_t add = s4 > 0 || part > 0 ? 1u : 0u;
                            if constexpr (Q8) mma_ts_x4<false>(s_at(i), qt, bv, id_s, add);
                            else mma_ss_x4<false>(s_at(i), av, bv, id_s, add);
                        }
                    }
                    mma_commit(smem_addr(&sh.s_full[slot][st]));
                    return true;
                };
                auto issue_pv = [&](int i, bool first) {
                    const int st = i % NS;
                    if (!mbar_wait(smem_addr(&sh.p_full[slot][i % NSB]), (i / NSB) & 1, abort, kWait)) return false;
                    if (Q8 && !mbar_wait(smem_addr(&sh.full_v[st]), (i / NS) & 1, abort, kWait)) return false;
                    tc_fence_after();
                    const uint64_t vb = sdesc(v_addr + st * C::KV_BYTES, 1024, C::SBO, C::LAYOUT);
                    // (both parts small, 2^-16 of the product: not taken)
#pragma unroll
                    for (int pp = 0; pp < (FINE ? 2 : 1); ++pp)
#pragma unroll
                        for (int part = 0; part < C::PARTS - pp || part == 0; ++part) {
                            if (part >= parts_of(i)) break;
                            uint32_t av[4];
                            uint64_t bv[4];
#pragma unroll
                            for (int s = 0; s < 4; ++s) {
                                av[s] = s_at(i) + (uint32_t)(s * 8 + pp * 32);
                                bv[s] = vb + (((uint32_t)s * 2u * C::SBO + part * C::PART_BYTES) >> 4);
                            }
                            mma_ts_x4<false>(tmem + (uint32_t)(slot * C::SLOT_COLS + C::O_COL), av, bv, id_o, first && part == 0 && pp == 0 ? 0u : 1u);
                        }
                    mma_commit(smem_addr(&sh.v_done[slot][st]));
                    return true;
                };
                // S(j + 1) goes over P(j - 1), whose product was issued before: the tensor pipe runs them in order.
                ok = ok && mbar_wait(smem_addr(&sh.q_ready[slot]), unit_no & 1, abort, kWait);
                ok = ok && issue_s(it);
                for (int i = 0; ok && i < n; ++i) {
                    if (i + 1 < n) ok = issue_s(it + i + 1);
                    if (slot > 0 && !tile_full(t0 + i))
                        ok = ok && mbar_wait(smem_addr(&sh.v_clean[(it + i) % NS]), ((it + i) / NS) & 1, abort, kWait);
                    ok = ok && issue_pv(it + i, i == 0);
                }
                if (!ok) *abort = 1;
            }
            it += n;
        } else {
            // ---- softmax: thread = row ----
            const int slot = warp >> 2, r = (warp & 3) * 32 + lane, row00 = row0 + slot * kTreeTileRows;
            const int rows = max(0, min(kTreeTileRows, rows_all - row00));
            const uint32_t lane_base = ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(slot * C::SLOT_COLS);
            uint8_t *sq = smem + slot * C::Q_BYTES;
            const int t = row_token(a, row00 + r);
            const bool on = r < rows && t < rq.n_nodes;
            // a warp without a row leaves P as it is: its products go to rows of O that nobody reads
            const bool live = __any_sync(0xffffffffu, on);
            // (units that the other row tile may still look at are at most NS back; this one's scan comes after every
            // warp's q_ready)
            if (threadIdx.x == 0) sh.bad[unit_no & 7] = 0;
            // this warp's query rows to shared memory (the last unit's products are done: its O was read)
            constexpr int U = D / 8;
            {
                const long long mine = (((long long)b * a.n_draft + t) * a.q_heads + g * a.group + (row00 + r) - t * a.group) * D;
                if constexpr (Q8) {
                    // to tensor memory: the converters' writes leave the shared memory no time to be read twice a product
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) {
                        uint32_t w[32];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const uint4 v = on ? *(const uint4 *)(a.q + mine + 64 * c + 8 * k) : make_uint4(0, 0, 0, 0);
                            w[4 * k] = v.x;
                            w[4 * k + 1] = v.y;
                            w[4 * k + 2] = v.z;
                            w[4 * k + 3] = v.w;
                        }
                        tmem_st32(tmem + lane_base + C::Q_COL + 32 * c, w);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                } else {
                    const uint32_t live = __ballot_sync(0xffffffffu, on);
#pragma unroll 16
                    for (int i = lane; i < 32 * U; i += 32) {
                        const int rr = i / U, uu = i % U;  // row of the warp (one per 32 or 16 lanes), unit
                        const long long row = __shfl_sync(0xffffffffu, mine, rr);
                        const bool has = (live >> rr) & 1u;
                        cp_async_16_or_zero(smem_addr(sq + bf16_off<D>((warp & 3) * 32 + rr, 8 * uu)), has ? a.q + row + 8 * uu : a.q, has);
                    }
                    cp_async_wait_all();
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&sh.q_ready[slot]));

            const ScoreFn score{a.scale_log2, a.cap_log2, a.cap_in};
            float m = -INFINITY;
            uint64_t l0 = 0, l1 = 0, lr = 0;  // the row's sum in four parts, and the rounded probabilities' in two
            bool draft_seen = false;
            unsigned long long word = ~0ull;
            for (int i = 0; i < n; ++i, ++it) {
                const int st = it % NS, par = (it / NS) & 1, j = t0 + i;
                const bool draft = j >= p_tiles;
                const int valid = draft ? rq.n_nodes : min(BN, rq.n_prefix - j * BN);
                if (draft) {
                    draft_seen = valid > 0;
                    word = !on ? 0ull
                           : a.ancestors ? __ldg(a.ancestors + (long long)b * a.n_draft + t)
                                         : (t >= 63 ? ~0ull : (2ull << t) - 1);
                }
                const bool full = tile_full(j);
                ok = ok && warp_wait(smem_addr(&sh.s_full[slot][st]), par, abort);
                if (!ok) break;
                tc_fence_after();
                const uint32_t s_col = tmem + lane_base + (uint32_t)(C::S_COL + (it % NSB) * BN);
                if (live) {
                    // the row's maximum of the tile
                    uint32_t sa[32], sb[32];
                    tmem_load32x2(s_col, s_col + 32, sa, sb);
                    bool sees = true;  // (a cap makes a score of an infinite product, which is no mask)
                    if (!full) {
                        const uint32_t bits = chunk_bits(word, 0, valid), bits1 = chunk_bits(word, 32, valid);
                        sees = (bits | bits1) != 0;
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            if (!((bits >> k) & 1u)) sa[k] = 0xff800000u;
                            if (!((bits1 >> k) & 1u)) sb[k] = 0xff800000u;
                        }
                    }
                    float top = -INFINITY, top1 = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        top = max3(top, __uint_as_float(sa[k]), __uint_as_float(sa[k + 1]));
                        top1 = max3(top1, __uint_as_float(sb[k]), __uint_as_float(sb[k + 1]));
                    }
                    top = fmaxf(top, top1);
                    const float mt = (CAP ? !sees : top == -INFINITY) ? -INFINITY : CAP ? score.capped(top) : top * a.scale_log2;
                    // m moves when the tile is more than 2^8 above it; O follows once P V(j - 1) has landed
                    const bool up = mt > m + 8.0f;
                    if (__any_sync(0xffffffffu, up)) {
                        const float f = up ? ex2(m - mt) : 1.0f;  // (0 for the first)
                        if (up) m = mt;
                        l0 = fma_pair(l0, pair_of(f, f), 0);
                        l1 = fma_pair(l1, pair_of(f, f), 0);
                        lr = fma_pair(lr, pair_of(f, f), 0);
                        if (i > 0) {
                            const int pst = (it - 1) % NS;
                            ok = warp_wait(smem_addr(&sh.v_done[slot][pst]), ((it - 1) / NS) & 1, abort);
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int c0 = 0; c0 < D; c0 += 32) {
                                uint32_t o[32];
                                tmem_load32(tmem + lane_base + C::O_COL + c0, o);
#pragma unroll
                                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                                tmem_st32(tmem + lane_base + C::O_COL + c0, o);
                            }
                            tmem_wait_st();
                        }
                    }
                    const float neg = m == -INFINITY ? 0.0f : -m;
                    const uint64_t scale2 = pair_of(a.scale_log2, a.scale_log2), neg2 = pair_of(neg, neg);
                    // (a masked score is -inf, of which the exponential is 0; a capped one is not, so it is put back to 0)
                    auto to_p = [&](uint32_t (&s)[32], uint32_t bits, uint32_t col) {
                        uint32_t p[16], rest[FINE ? 16 : 1];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float2 v = make_float2(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1]));
                            if (CAP) v = make_float2(score.capped(v.x) + neg, score.capped(v.y) + neg);
                            else v = of_pair(fma_pair(pair_of(v.x, v.y), scale2, neg2));
                            v = make_float2(ex2(v.x), ex2(v.y));
                            if (CAP && !full) {
                                if (!((bits >> (2 * k)) & 1u)) v.x = 0.0f;
                                if (!((bits >> (2 * k + 1)) & 1u)) v.y = 0.0f;
                            }
                            if (k & 1) l1 = add_pair(l1, pair_of(v.x, v.y));
                            else l0 = add_pair(l0, pair_of(v.x, v.y));
                            p[k] = pack_bf16(v.x, v.y);
                            const uint64_t hi = pair_of(__uint_as_float(p[k] << 16), __uint_as_float(p[k] & 0xffff0000u));
                            if constexpr (FINE) {
                                const float2 r = of_pair(fma_pair(hi, pair_of(-1.0f, -1.0f), pair_of(v.x, v.y)));
                                rest[k] = pack_bf16(r.x, r.y);
                            } else {
                                lr = add_pair(lr, hi);
                            }
                        }
                        tmem_st16(col, p);
                        if constexpr (FINE) tmem_st16(col + 32, rest);
                    };
                    to_p(sa, full ? 0xffffffffu : chunk_bits(word, 0, valid), s_col);
                    to_p(sb, full ? 0xffffffffu : chunk_bits(word, 32, valid), s_col + 16);
                    tmem_wait_st();
                }
                if (!full && slot == 0) {  // rows past the last key hold whatever was there: 0 * that must be 0
                    ok = warp_wait(smem_addr(Q8 ? &sh.full_v[st] : &sh.full[st]), par, abort);
                    if (!ok) break;
                    uint8_t *vt = smem + C::OFF_V + st * C::KV_BYTES;
                    for (int e = max(0, valid) * U + threadIdx.x; e < BN * U; e += 128)
                        *(uint4 *)(vt + bf16_off<D>(e / U, (e % U) * 8)) = make_uint4(0, 0, 0, 0);
                    // Drafted values that are not finite leave the tile: 0 * inf would reach rows that may not
                    // see them. Rows that do get them at the end.
                    for (int e = threadIdx.x; draft && e < valid * U; e += 128) {
                        uint16_t *w = (uint16_t *)(vt + bf16_off<D>(e / U, (e % U) * 8));
                        const uint4 v = *(const uint4 *)w;
                        const uint32_t ww[4] = {v.x, v.y, v.z, v.w};
                        bool any = false;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            any = any || (ww[k] & 0x7f80u) == 0x7f80u || (ww[k] & 0x7f800000u) == 0x7f800000u;
                        if (any) {
                            atomicOr(&sh.bad[unit_no & 7], 1ull << (e / U));
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if ((w[k] & 0x7f80u) == 0x7f80u) w[k] = 0;
                        }
                    }
                    fence_proxy_async();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_addr(&sh.p_full[slot][it % NSB]));
                    if (RT == 2 && slot == 0) mbar_arrive(smem_addr(&sh.v_clean[st]));
                }
            }
            if (ok && n > 0) {
                ok = warp_wait(smem_addr(&sh.v_done[slot][(it - 1) % NS]), ((it - 1) / NS) & 1, abort);
                tc_fence_after();
            }
            if (!ok) *abort = 1;
            if (ok) {
                const bool whole = t0 == 0 && t1 == n_tiles;
                const long long part = (2ll * blockIdx.x + (t0 == 0 ? 1 : 0)) * ROWS + slot * kTreeTileRows;
                const float2 la = of_pair(l0), lb = of_pair(l1), lc = of_pair(lr);
                const float l = (la.x + lb.x) + (la.y + lb.y), lrow = FINE ? l : lc.x + lc.y;
                const float f = !whole ? 1.0f : lrow == 0.0f ? 0.0f : 1.0f / lrow;
                const int hq = g * a.group + (row00 + r) - t * a.group;
                const long long at = ((long long)b * a.n_draft + t) * a.q_heads + hq;
                if (r < rows) {
                    if (!whole) a.ws_ml[part + r] = on ? make_float4(m, l, lrow, 0.0f) : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
                    else if (a.lse) a.lse[at] = on && l != 0.0f ? (m + __log2f(l)) * 0.6931471805599453f : -INFINITY;
                }
                const unsigned long long bad = draft_seen ? sh.bad[unit_no & 7] : 0ull;
                const uint32_t p_col = tmem + lane_base + C::S_COL + (uint32_t)(((it - 1) % NSB) * BN);
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t o[32];
                    tmem_load32(tmem + lane_base + C::O_COL + c0, o);
                    // rare: drafted values that are not finite, for the rows that see them (the drafts are the
                    // unit's last tile, so their P is still there)
                    for (unsigned long long rest = bad; rest; rest &= rest - 1) {
                        const int k = __ffsll((long long)rest) - 1;
                        uint32_t pair;
                        asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
                                     : "=r"(pair)
                                     : "r"(p_col + (uint32_t)(k >> 1))
                                     : "memory");
                        const float p = bf16_bits_to_f32((uint16_t)(k & 1 ? pair >> 16 : pair));
                        const uint16_t *v = a.v_draft + kv_row + (long long)k * hk * D + c0;
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float y = bf16_bits_to_f32(__ldg(v + e));
                            if (!isfinite(y) && ((word >> k) & 1ull)) o[e] = __float_as_uint(fmaf(p, y, __uint_as_float(o[e])));
                        }
                    }
                    // a row without a key has nothing (not 0 * what the columns hold)
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = on && l != 0.0f ? __float_as_uint(__uint_as_float(o[e]) * f) : 0u;
                    // through the warp's query rows, which are done with, so that whole rows of 128 bytes are
                    // written: unit k of row i lies at unit k ^ (i & 7) of 128 bytes
                    uint8_t *stage = sq + (warp & 3) * 32 * D * 2;
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        *(uint4 *)(stage + lane * 128 + ((k ^ (lane & 7)) << 4)) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                    __syncwarp();
                    const int unit = lane & 7;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int i = 4 * k + (lane >> 3), rr = (warp & 3) * 32 + i;
                        const uint4 v = *(const uint4 *)(stage + i * 128 + ((unit ^ (i & 7)) << 4));
                        const long long row = __shfl_sync(0xffffffffu, at, i);
                        if (rr >= rows) continue;
                        if (!whole) {
                            *(uint4 *)(a.ws_o + (part + rr) * D + c0 + 4 * unit) = v;
                        } else if (a.out_dtype == EKV_DTYPE_F32) {
                            *(uint4 *)((float *)a.out + row * D + c0 + 4 * unit) = v;
                        } else {
                            *(uint2 *)((uint16_t *)a.out + row * D + c0 + 4 * unit) =
                                make_uint2(pack_bf16(__uint_as_float(v.x), __uint_as_float(v.y)), pack_bf16(__uint_as_float(v.z), __uint_as_float(v.w)));
                        }
                    }
                    __syncwarp();
                }
                tc_fence_before();
            }
        }
        ++unit_no;
        x += n;
    }
    if (!ok && lane == 0) report_error(a.pool.status, DEV_ERR_TIMEOUT, blockIdx.x, warp, 11);
    if (warp == C::FEED_WARP && !ok && lane == 0) {
        for (int i = 0; i < (Q8 ? C::NR : NS); ++i) {  // leave no copy writing this CTA's shared memory
            const uint32_t bar = smem_addr(Q8 ? &sh.raw_full[i] : &sh.full[i]);
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

template <int D, int RT, bool Q8, bool CAP, bool FINE>
int launch_form(const TreeArgs &a, int grid, cudaStream_t s) {
    using C = TCfg<D, RT, Q8>;
    static std::atomic<uint64_t> done{0};
    if (const int rc = allow_smem(tree_tile_kernel<D, RT, Q8, CAP, FINE>, C::SMEM, done)) return rc;
    return launch_after(tree_tile_kernel<D, RT, Q8, CAP, FINE>, grid, C::THREADS, C::SMEM, s, a);
}

template <int D, int RT, bool Q8 = false>
int launch(const TreeArgs &a, int grid, cudaStream_t s) {
    if (a.out_dtype == EKV_DTYPE_F32)
        return a.cap_log2 != 0.0f ? launch_form<D, RT, Q8, true, true>(a, grid, s) : launch_form<D, RT, Q8, false, true>(a, grid, s);
    return a.cap_log2 != 0.0f ? launch_form<D, RT, Q8, true, false>(a, grid, s) : launch_form<D, RT, Q8, false, false>(a, grid, s);
}

}  // namespace

// Where this form begins, measured over pools of 800 to 4096 keys and 1 to 16 requests. Scores without a cap: from 17
// rows of a KV head (16 requests of 4096 keys, 8 KV heads: 24 rows 71 -> 46 us at head_dim 64, 90 -> 69 at 128, 131 -> 80
// at 256; with 16 rows the rows kernel is ahead, 62 against 67 at head_dim 128). A cap costs a thread 64 tanhf a tile here,
// which the rows kernel spreads over all lanes: from 33 rows (head_dim 128: 24 rows 103 against 119 us, 48 rows 170
// against 116), and from 65 at head_dim 64 (48 rows: 25 against 24 us in a middling call, but 20 against 25 with 39 ragged
// ones). Q8_0 at head_dim 64 and 128, the same calls: 32 rows 102 -> 97 and 172 -> 152 us, 256 rows 505 -> 184 and
// 826 -> 297; with a cap from 65 (head_dim 128: 48 rows 258 against 323 us, 256 rows 957 against 591). At head_dim 256 two
// parts of K and V do not fit the shared memory.
int tree_tile_rows(const PoolView &p, int rows, bool capped) {
    const int below = !capped ? 16 : p.head_dim == 64 || p.dtype == EKV_DTYPE_Q8_0 ? 64 : 32;
    if (rows <= below) return 0;
    if (p.dtype != EKV_DTYPE_BF16) return p.head_dim == 64 || p.head_dim == 128 ? kTreeTileRows : 0;
    if (p.head_dim == 64 || p.head_dim == 128) return rows > kTreeTileRows ? 2 * kTreeTileRows : kTreeTileRows;
    return p.head_dim == 256 ? kTreeTileRows : 0;
}

int tree_tile_ctas(const PoolView &p, int rows, int sms) {
    return sms * (p.dtype == EKV_DTYPE_BF16 && p.head_dim <= 128 && rows <= kTreeTileRows ? 2 : 1);
}

int launch_tree_tile(const TreeArgs &a, int grid, cudaStream_t s) {
    if (a.pool.dtype == EKV_DTYPE_Q8_0) {
        switch (a.pool.head_dim) {
            case 64: return launch<64, 1, true>(a, grid, s);
            case 128: return launch<128, 1, true>(a, grid, s);
            default: return EKV_ERR_UNSUPPORTED;
        }
    }
    const bool two = a.n_draft * a.group > kTreeTileRows;
    switch (a.pool.head_dim) {
        case 64: return two ? launch<64, 2>(a, grid, s) : launch<64, 1>(a, grid, s);
        case 128: return two ? launch<128, 2>(a, grid, s) : launch<128, 1>(a, grid, s);
        case 256: return launch<256, 1>(a, grid, s);
        default: return EKV_ERR_UNSUPPORTED;
    }
}

}  // namespace ekv
