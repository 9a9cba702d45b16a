// ekv_window_tile.cu -- windowed attention of many rows per KV head (prompts, chunks) on tcgen05.
//
// out = sum_k p_k v_k / sum_k p_k with p_k = exp(scale q.k - m) over the keys a row sees (ekv_window.cuh), m a running reference that
// moves only when a score is 2^24 (8-bit pages: 2^8) above it. S = Q K^T with both operands in shared memory and S in tensor memory, P in
// 16 bits over S's own columns, O += P V with P read from tensor memory. P is rounded to bf16 (bf16 pages) and the row divided by the
// sum of the rounded ones; over 8-bit pages operands are f16 (a value's int8 times its scale keeps 11 bits, P too, down to 2^-21 of the
// row's largest; below that its steps are 2^-31 of it).
//
// Roles of a CTA's warps, each in step with the CTA's tiles by its own count: feed (K, V), convert (8-bit pages, K and V apart) or
// look_at_values (bf16), products (a warp per row tile), softmax (a thread per row; head_dim 256: two). What bounds it: a row
// tile's chain of scores, maximum, exponentials, P, next products. Two row tiles fill it for the special-function unit (1024 of a
// 64-key tile's 2450 cycles) and the tensor pipe (1300 of them); a unit's end and beginning take 9000 cycles, beside the 15
// tiles that a unit of the eight prompts below has a fifth.
// 32 / 8 heads of 128: a prompt of 16384 tokens 2284 us (963 TFLOP/s of the products that rows see, 57% of a measured bf16 product), over
// 8-bit pages 2607; 8 prompts of up to 4096, window 1024 and 4 first tokens: 625 us (638), over 8-bit pages 769. 8 / 1 heads of 256, 8192
// tokens: 297 us (926). At 1965 MHz: after a second of such calls the power limit leaves 1.8 GHz, and the eight prompts take 683.
// Measured and left out, with the first prompt's and the eight's times, which were 2335 and 637 us then: 128 keys a tile with one S tile
// 2386 and 773; two warps to a row in place of one for head_dim 128 2654 and 718 (for 256, where one row tile leaves the schedulers a
// warp each, 343 instead of 396); a part of the exponentials by polynomial 2333 and 645 (an eighth), 2448 and 711 (a quarter).

#include "ekv_window.cuh"

namespace ekv {
namespace {

using namespace decode;
using namespace sm100;
using namespace window;

constexpr int kTileRows = 128;  // rows of a row tile: the lanes of tensor memory

// head_dim 64 and 128: two row tiles (slots) of a KV head share an SM and each K/V tile; head_dim 256: one, as two outputs do not fit the
// tensor memory. A slot has two S tiles, so that the scores of the next tile are there when the exponentials of one are done.
template <int D, bool Q8>
struct WCfg {
    static constexpr int RT = D > 128 ? 1 : 2;
    static constexpr int BN = 64;                     // keys per tile
    static constexpr int NSB = 2;                     // S tiles of a row tile
    // K and V stages. 8-bit pages: one (two), as they are filled from the blocks as stored, which have room to be on their way instead
    static constexpr int NS = D <= 128 ? (Q8 ? 2 : 4) : (Q8 ? 1 : 2);
    static constexpr int NSF = NS > NSB ? NS : NSB;   // barriers of S: a tile's S may be done while S of the one before is not read
    // a reference that is 2^LIMIT too low does not move: P and what is summed are floating point numbers, and only their range counts
    static constexpr float LIMIT = Q8 ? 8.0f : 24.0f;
    // f16 ends at 2^16 and has steps of 2^-24 below 2^-14: P is 2^HEADROOM times what it stands for, as its sum is, so that a key is off by
    // 2^-32 of its row's largest at most and not by 2^-25 (one heavy key before 60 000 light ones, 26 bits below it: those were lost)
    static constexpr float HEADROOM = Q8 ? 7.0f : 0.0f;
    static_assert(!Q8 || LIMIT + HEADROOM < 16.0f, "P in f16");
    static constexpr uint32_t SBO = 16 * D, LAYOUT = 2;
    static constexpr int KV_BYTES = BN * D * 2, Q_BYTES = kTileRows * D * 2;
    static constexpr int NR = D > 128 ? 2 : 4, RAW = BN * D + BN * (D / 32) * 2;  // Q8: tiles of K, and of V, as they are stored
    static constexpr int S_COL = 0, O_COL = BN * NSB, SLOT_COLS = 256, COLS = 512;
    static constexpr int OFF_K = RT * Q_BYTES, OFF_V = OFF_K + NS * KV_BYTES, OFF_RAW = OFF_V + NS * KV_BYTES;
    static constexpr int OFF_SH = OFF_RAW + (Q8 ? (2 * NR * RAW + 1023) / 1024 * 1024 : 0);
    static constexpr int OFF_X = OFF_SH + 2048, OFF_BAD = OFF_X + RT * 2 * kTileRows * 4, SHARED = OFF_BAD - OFF_SH + (Q8 ? 0 : 8192);
    static constexpr int SMEM = OFF_SH + SHARED + 1024;
    static constexpr int SHARE = RT == 1 ? 2 : 1;  // softmax warps of 32 rows
    static constexpr int ROW_WARPS = 4 * SHARE * RT, MMA_WARP = ROW_WARPS, FEED_WARP = MMA_WARP + RT;
    // K's feeder, V's feeder; bf16: four warps that look at V; Q8: four that convert K, four that convert V
    static constexpr int SCRUB_WARP = FEED_WARP + 2, SCRUB_WARPS = 4, CONV_WARP = FEED_WARP + 2, CONV_WARPS = 4;
    static constexpr int WARPS = Q8 ? CONV_WARP + 2 * CONV_WARPS : SCRUB_WARP + SCRUB_WARPS, THREADS = WARPS * 32;
    // 8-bit pages, two row tiles: 20 warps leave 96 registers to a thread at launch, and a row's 64 scores take more. (The compiler allots
    // 96 to all and spills 130 words, whatever the row warps raise themselves to. With two warps in place of four for each conversion
    // there is room for 128; 16384 tokens of head_dim 128 then took 2960 us instead of 2620.)
    static constexpr bool SPLIT_REGS = Q8 && RT == 2;
    static constexpr int ROW_REGS = 136, OTHER_REGS = 64;
    static_assert(!SPLIT_REGS || (THREADS == 640 && 256 * ROW_REGS + 384 * OTHER_REGS <= 640 * 96), "registers");
    static_assert(O_COL + D <= (RT == 2 ? SLOT_COLS : COLS) && SMEM <= 232448, "tensor memory, shared memory");
};

constexpr int kBadChunks = 56;  // four for each tile that only some rows of a unit see: at most 13 for 256 tokens (five around their own
                                // slots, six around the window's end, one each where the first tokens and the keys end)
constexpr int kBadUnits = 16;   // V is looked at no more than the stages' four tiles ahead of the rows, by four warps that are no more than
                                // that apart: the unit eight on may be made empty

// Where a CTA's range of a split call begins, and where it ends (Units).
struct RangeStart {
    int b, g, rt;      // the unit that holds place x
    uint32_t at;       // its first place
    uint32_t x, hi, total;
    int ctas;
};

struct WShared {
    uint64_t full_k[4], full_v[4];       // K, V of the stage are there
    uint64_t raw_full[2][4], raw_empty[2][4];  // Q8: [K, V] a tile has landed; is converted
    uint64_t s_full[2][4];               // [slot][tile % NSF] S done
    uint64_t v_free[4];                  // both slots' P V done, and (bf16) the tile looked at
    uint64_t p_full[2][2];               // [slot][S tile] P written
    uint64_t q_ready[2], o_done[2], drained[2];
    uint64_t turn[2];                    // [slot] it may issue its next group of products
    uint64_t v_clean[4];                 // V of a tile that only some rows see holds finite values
    uint32_t tmem;
    int abort;
    RangeScratch range;
    RangeStart start;
    int unfit[8];  // Q8: [converting warp] some tile's scales do not fit
};

// [unit % kBadUnits] keys whose values are not all finite, 32 to an entry
struct WBad {
    int n[kBadUnits];
    uint32_t keys[kBadUnits][kBadChunks];
    int first[kBadUnits][kBadChunks];
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// The two warps that share rows (named barrier id): any of their lanes' x; both there.
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

// One lane of a converged warp. With `lane == 0` in its place the compiler guards each tcgen05.mma by itself against lanes that
// differ: 80 to 110 cycles an instruction, more than most of them run, so that issuing bound the kernel.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ void tmem_load8(uint32_t at, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at)
                 : "memory");
}

// Lane i of four has unit k of row i in x[k], and gets unit i of row k: four rows' 64 bytes each in one store of the four lanes.
__device__ __forceinline__ void transpose4(uint4 (&x)[4], int lane) {
    auto swap = [&](uint4 &a, uint4 &b, int m) {  // the upper lane's a for the lower one's b
        const bool up = lane & m;
        uint4 give = up ? a : b;
        give.x = __shfl_xor_sync(0xffffffffu, give.x, m);
        give.y = __shfl_xor_sync(0xffffffffu, give.y, m);
        give.z = __shfl_xor_sync(0xffffffffu, give.z, m);
        give.w = __shfl_xor_sync(0xffffffffu, give.w, m);
        (up ? a : b) = give;
    };
    swap(x[0], x[1], 1);
    swap(x[2], x[3], 1);
    swap(x[0], x[2], 2);
    swap(x[1], x[3], 2);
}

__device__ __forceinline__ bool scale_fits(uint16_t bits) { return fabsf(f16_bits_to_f32(bits)) <= 515.0f; }

// The blocks' int8 rows as f16 values, rounded once; rows past `valid` are zero. Values whose scale leaves the f16 range with them are 0;
// false where there are any.
template <int D, int ROWS, int THREADS>
__device__ __forceinline__ bool convert_tile(const uint8_t *raw, uint8_t *dst, int valid, int thread) {
    constexpr int U = D / 16;
    bool fits = true;
#pragma unroll 4
    for (int e = thread; e < ROWS * U; e += THREADS) {
        // four 16-byte columns and two rows in every eight lanes, which then write to eight different columns of the swizzled rows
        const int rest = e >> 3, u = (rest % (U / 4)) * 4 + (e & 3), row = rest / (U / 4) * 2 + ((e >> 2) & 1);
        uint32_t out[8] = {};
        if (row < valid) {
            const uint4 v = *(const uint4 *)(raw + q8_qs_off(row, 16 * u, D));
            const uint16_t bits = *(const uint16_t *)(raw + ROWS * D + (row * (D / 32) + (u >> 1)) * 2);
            const bool ok = scale_fits(bits);
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
            *(uint4 *)(dst + bf16_off<D>(row, 16 * u + 8 * k)) = make_uint4(out[4 * k], out[4 * k + 1], out[4 * k + 2], out[4 * k + 3]);
    }
    return fits;
}

// ---- the units of a CTA, in the same order in every warp ----
// kCutUnits: the range [x, hi) of all tiles in the order request, KV head, row tile, tile, where a unit counts kUnitCost tiles more for
// what it costs beside them (query rows, the first tile's way, the end): without that the CTA of a long prompt's first rows took half
// as long again (8192 tokens of head_dim 256: 367 us at 2, 294 at 4, 300 at 8). The row tiles of a head follow one another, so that a CTA
// finds most of a window in L2: with the heads innermost the windows of all CTAs' heads did not fit it.
// kWholeUnits: the same ranges, but a unit belongs to the CTA whose range its middle is in.
// Else whole units, the longest (a request's last rows) first, back and forth over the CTAs.
constexpr int kUnitCost = kWindowUnitCost;
template <int ROWS, int BN>
struct Units {
    int rt, round;     // row tile (split); rounds over the CTAs so far
    uint32_t at, x, hi;
    int b, g, row0;    // the unit: request, KV head, first row
    int rq_of;         // the request that rq describes
    WinReq rq;
    int n_tiles, t0, t1;  // its tiles, and this CTA's
    static __device__ __forceinline__ int tiles_of(const WindowArgs &a, const WinReq &r, int rt) {
        const int row0 = rt * ROWS;
        if (row0 >= r.n * a.group) return 0;
        const Span sp(a, r, row_token(a, row0), last_token(a, row0, ROWS, r.n));
        return max(1, (sp.keys + BN - 1) / BN);
    }
    static __device__ __forceinline__ uint32_t cost_of(const WindowArgs &a, const WinReq &r, int rt) {
        const int n = tiles_of(a, r, rt);
        return n > 0 ? (uint32_t)(n + kUnitCost) : 0u;
    }
    __device__ __forceinline__ Units(const RangeStart &s) : rt(s.rt), round(0), at(s.at), x(s.x), hi(s.hi), b(s.b), g(s.g), rq_of(-1) {}
    __device__ __forceinline__ bool next(const WindowArgs &a, bool report) {
        const int hk = a.pool.kv_heads;
        if (a.split) {
            while ((x < hi || a.split == kWholeUnits) && b < a.n_batch) {
                if (rq_of != b) rq = load_win_req(a, b, false), rq_of = b;
                n_tiles = tiles_of(a, rq, rt);
                if (n_tiles == 0) {  // the request has no more rows: its next head, or the next request
                    rt = 0;
                    if (++g == hk || rq.n == 0) {
                        g = 0;
                        ++b;
                    }
                    continue;
                }
                const uint32_t cost = (uint32_t)(n_tiles + kUnitCost);
                if (x >= at + cost) {
                    at += cost;
                    ++rt;
                    continue;
                }
                if (a.split == kWholeUnits) {
                    // those whose middle is in the range
                    const uint32_t middle = at + cost / 2;
                    if (middle >= hi) return false;
                    if (middle < x) {
                        x = at + cost;
                        continue;
                    }
                    x = at + cost;
                    row0 = rt * ROWS;
                    t0 = 0;
                    t1 = n_tiles;
                    return true;
                }
                const int from = (int)(x - at), to = (int)min(cost, from + (hi - x));
                x += to - from;
                t0 = max(0, from - kUnitCost);
                t1 = to - kUnitCost;
                row0 = rt * ROWS;
                if (t1 > t0) return true;  // (not only what a unit costs beside its tiles)
            }
            return false;
        }
        const int all = a.n_batch * a.row_tiles * hk;  // (below 2^31: checked at the launch)
        for (;;) {
            const long long from = (long long)round * gridDim.x, place = from + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
            if (from >= all) return false;
            ++round;
            if (place >= all) continue;
            const int rest = (int)place / hk, k = rest / a.n_batch;
            rt = a.row_tiles - 1 - k;
            g = (int)place - rest * hk;
            b = rest - k * a.n_batch;
            rq = load_win_req(a, b, report && rt == 0 && g == 0);
            n_tiles = tiles_of(a, rq, rt);
            if (n_tiles == 0) continue;
            row0 = rt * ROWS;
            t0 = 0;
            t1 = n_tiles;
            return true;
        }
    }
    __device__ __forceinline__ int rows(const WindowArgs &a) const { return min(ROWS, rq.n * a.group - row0); }
    __device__ __forceinline__ Span span(const WindowArgs &a) const {
        return Span(a, rq, row_token(a, row0), last_token(a, row0, ROWS, rq.n));
    }
};

template <int D, bool Q8>
__device__ __forceinline__ bool feed(const WindowArgs &a, uint8_t *smem, WShared &sh, Units<WCfg<D, Q8>::RT * kTileRows, WCfg<D, Q8>::BN> u) {
    using C = WCfg<D, Q8>;
    constexpr int BN = C::BN, NS = C::NS, RT = C::RT;
    volatile int *abort = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = a.pool.kv_heads;
    bool ok = true;
    const bool is_v = warp != C::FEED_WARP;
    int it = 0;  // tiles of this CTA so far
    while (u.next(a, false)) {
        const Span sp = u.span(a);
        // ---- feeders ----
        auto want = [](int, int) {};
        auto block = [&](int e) { return lookup_block(a.pool, u.rq.seq, e); };
        const int64_t v_from_k = (int64_t)hk * a.pool.tile_bytes;
        if constexpr (!Q8) {
            Run next = find_run<BN>(a, sp, u.g, u.t0 * BN, lane, want, block);
            for (int j = u.t0; j < u.t1; ++j, ++it) {
                const int st = it % NS, par = (it / NS) & 1;
                const Run r = next;
                if (j + 1 < u.t1) next = find_run<BN>(a, sp, u.g, (j + 1) * BN, lane, want, block);
                if (it >= NS) {
                    if (is_v) ok = ok && warp_wait(smem_addr(&sh.v_free[st]), par ^ 1, abort);
#pragma unroll
                    for (int k = 0; k < RT; ++k)
                        if (!is_v) ok = ok && warp_wait(smem_addr(&sh.s_full[k][(it - NS) % C::NSF]), ((it - NS) / C::NSF) & 1, abort);
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
            Run next = find_run<BN>(a, sp, u.g, u.t0 * BN, lane, want, block);
            for (int j = u.t0; j < u.t1; ++j, ++it) {
                const int rs = it % C::NR;
                const Run r = next;
                if (j + 1 < u.t1) next = find_run<BN>(a, sp, u.g, (j + 1) * BN, lane, want, block);
                if (it >= C::NR) ok = ok && warp_wait(smem_addr(&sh.raw_empty[is_v][rs]), (it / C::NR - 1) & 1, abort);
                if (!ok) {
                    *abort = 1;
                    continue;
                }
                const uint32_t dst = smem_addr(smem + C::OFF_RAW + (is_v * C::NR + rs) * C::RAW), bar = smem_addr(&sh.raw_full[is_v][rs]);
                const uint32_t bytes = r.src ? (uint32_t)(r.n * (D + D / 16)) : 0u, all = __reduce_add_sync(0xffffffffu, bytes);
                if (lane == 0) mbar_arrive_expect_tx(bar, all);
                __syncwarp();
                if (!r.src) continue;
                const uint8_t *src = r.src + (is_v ? v_from_k : 0);
                bulk_g2s(dst + r.row * D, src + r.rib * D, (uint32_t)(r.n * D), bar);
                bulk_g2s(dst + BN * D + r.row * (D / 16), src + (int64_t)a.pool.block_tokens * D + r.rib * (D / 16), (uint32_t)(r.n * (D / 16)), bar);
            }
        }
    }
    if (!ok && lane == 0) {
        // leave no copy writing this CTA's shared memory
        for (int i = 0; i < (Q8 ? C::NR : NS); ++i) {
            const uint32_t bar = smem_addr(Q8 ? &sh.raw_full[is_v][i] : is_v ? &sh.full_v[i] : &sh.full_k[i]);
            mbar_wait_drain(bar, 0, kWait / 64);
            mbar_wait_drain(bar, 1, kWait / 64);
        }
    }
    return ok;
}

// Whether the scales that the rows of this CTA's units see fit, one lane a key. Asked once some tile's did not: tiles hold up to 14 rows
// that no row sees. (Told apart where a tile is converted, they cost 2 to 4% of a prompt; here, less than 1%.)
template <int D, class U>
__device__ __forceinline__ bool seen_scales_fit(const WindowArgs &a, U u, int bn, int lane) {
    const PoolView &p = a.pool;
    bool fits = true;
    while (u.next(a, false)) {
        const Span sp = u.span(a);
        const int hidden = sp.hidden(a), n_hidden = sp.n_hidden(a), end = min(u.t1 * bn, sp.keys);
#pragma unroll 1
        for (int key = u.t0 * bn + lane; key < end; key += 32) {
            if ((uint32_t)(key - hidden) < (uint32_t)n_hidden) continue;
            const int slot = sp.slot(key), e = slot / p.block_tokens, blk = lookup_block(p, u.rq.seq, e);
            if (blk < 0) continue;
#pragma unroll 1
            for (int i = 0; i < 2 * (D / 32); ++i) {
                const uint8_t *tile = p.prefix + prefix_tile_index(p, a.layer, blk, i & 1, u.g) * p.tile_bytes;
                fits = fits && scale_fits(((const uint16_t *)(tile + (int64_t)p.block_tokens * D))[(slot - e * p.block_tokens) * (D / 32) + (i >> 1)]);
            }
        }
    }
    return __all_sync(0xffffffffu, fits);
}

template <int D, bool Q8>
__device__ __forceinline__ bool convert(const WindowArgs &a, uint8_t *smem, WShared &sh, Units<WCfg<D, Q8>::RT * kTileRows, WCfg<D, Q8>::BN> u) {
    using C = WCfg<D, Q8>;
    constexpr int BN = C::BN, NS = C::NS, RT = C::RT;
    volatile int *abort = &sh.abort;
    const int lane = threadIdx.x & 31, thread = threadIdx.x - C::CONV_WARP * 32, is_v = thread >= C::CONV_WARPS * 32;
    bool ok = true;
    int it = 0;  // tiles of this CTA so far
    bool fits = true;
    while (u.next(a, false)) {
        const Span sp = u.span(a);
        for (int j = u.t0; j < u.t1; ++j, ++it) {
            const int st = it % NS, rs = it % C::NR;
            if (it >= NS) {  // the stage is free
                if (is_v) ok = ok && warp_wait(smem_addr(&sh.v_free[st]), (it / NS - 1) & 1, abort);
#pragma unroll
                for (int k = 0; k < RT; ++k)
                    if (!is_v) ok = ok && warp_wait(smem_addr(&sh.s_full[k][(it - NS) % C::NSF]), ((it - NS) / C::NSF) & 1, abort);
            }
            ok = ok && warp_wait(smem_addr(&sh.raw_full[is_v][rs]), (it / C::NR) & 1, abort);
            if (!ok) {
                *abort = 1;
                continue;
            }
            fits &= convert_tile<D, BN, C::CONV_WARPS * 32>(smem + C::OFF_RAW + (is_v * C::NR + rs) * C::RAW, smem + (is_v ? C::OFF_V : C::OFF_K) + st * C::KV_BYTES,
                                                           sp.keys - j * BN, thread & (C::CONV_WARPS * 32 - 1));
            fence_proxy_async();  // read by the tensor core; the next blocks come through the copy engine
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_addr(&sh.raw_empty[is_v][rs]));
                mbar_arrive(smem_addr(is_v ? &sh.full_v[st] : &sh.full_k[st]));
            }
        }
    }
    fits = __all_sync(0xffffffffu, fits);
    if (lane == 0) sh.unfit[thread / 32] = !fits;  // (no word to clear: a store more at the kernel's start took 1.6% of eight windowed prompts)
    return ok;
}

template <int D, bool Q8>
__device__ __forceinline__ bool look_at_values(const WindowArgs &a, uint8_t *smem, WShared &sh, Units<WCfg<D, Q8>::RT * kTileRows, WCfg<D, Q8>::BN> u) {
    using C = WCfg<D, Q8>;
    constexpr int BN = C::BN, NS = C::NS;
    volatile int *abort = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    bool ok = true;
    int it = 0;  // tiles of this CTA so far
    int unit_no = 0;
    while (u.next(a, false)) {
        const Span sp = u.span(a);
        auto unit_sees = [&](int j) { return sp.all_see(a, j * BN, BN); };
        // ---- values that are not finite leave the tiles that only some rows see: 0 * inf would reach the others ----
        WBad &found = *(WBad *)(smem + C::OFF_BAD);
        const int ub = unit_no % kBadUnits;
        if (warp == C::SCRUB_WARP && lane == 0) found.n[(unit_no + kBadUnits / 2) % kBadUnits] = 0;
        for (int j = u.t0; j < u.t1; ++j, ++it) {
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
            // a warp takes BN / 4 keys, a lane up to eight units of them at a time
            uint8_t *vt = smem + C::OFF_V + st * C::KV_BYTES;
            constexpr int U = D / 8, KEYS = BN / C::SCRUB_WARPS, PER = KEYS * U / 32, STEP = PER < 8 ? PER : 8;
            static_assert(PER % STEP == 0 && KEYS <= 32 && KEYS * U % 32 == 0, "whole steps inside the warp's keys");
            const int first = (warp - C::SCRUB_WARP) * KEYS, valid = min(BN, sp.keys - j * BN);
            uint32_t bad = 0;
#pragma unroll 1
            for (int e0 = 0; e0 < PER; e0 += STEP) {
                uint4 v[STEP];
#pragma unroll
                for (int e = 0; e < STEP; ++e) {
                    const int i = (e0 + e) * 32 + lane;
                    v[e] = *(const uint4 *)(vt + bf16_off<D>(first + i / U, (i % U) * 8));
                }
#pragma unroll
                for (int e = 0; e < STEP; ++e) {
                    const int i = (e0 + e) * 32 + lane, r = first + i / U;
                    uint32_t w[4] = {v[e].x, v[e].y, v[e].z, v[e].w};
                    bool any = false;
#pragma unroll
                    for (int k = 0; k < 4; ++k) any = any || (w[k] & 0x7f80u) == 0x7f80u || (w[k] & 0x7f800000u) == 0x7f800000u;
                    if (r < valid && !any) continue;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if ((w[k] & 0x7f80u) == 0x7f80u || r >= valid) w[k] &= 0xffff0000u;
                        if ((w[k] & 0x7f800000u) == 0x7f800000u || r >= valid) w[k] &= 0xffffu;
                    }
                    if (r < valid) bad |= 1u << (r - first);
                    *(uint4 *)(vt + bf16_off<D>(r, (i % U) * 8)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            bad = __reduce_or_sync(0xffffffffu, bad);
            if (bad && lane == 0) {
                const int i = atomicAdd(&found.n[ub], 1);
                if (i < kBadChunks) {
                    found.keys[ub][i] = bad;
                    found.first[ub][i] = j * BN + first;
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_addr(&sh.v_clean[st]));
                mbar_arrive(smem_addr(&sh.v_free[st]));
            }
        }
        ++unit_no;
    }
    return ok;
}

template <int D, bool Q8>
__device__ __forceinline__ bool products(const WindowArgs &a, uint8_t *smem, WShared &sh, Units<WCfg<D, Q8>::RT * kTileRows, WCfg<D, Q8>::BN> u, uint32_t tmem) {
    using C = WCfg<D, Q8>;
    constexpr int BN = C::BN, NS = C::NS, NSB = C::NSB, RT = C::RT;
    volatile int *abort = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    bool ok = true;
    int it = 0, live_units = 0;  // tiles of this CTA so far; units that this slot had rows for
    [[maybe_unused]] int turns = 0;
    [[maybe_unused]] uint32_t clean_phase = 0;  // v_clean, a bit per stage
    while (u.next(a, false)) {
        const int n = u.t1 - u.t0;
        const Span sp = u.span(a);
        auto unit_sees = [&](int j) { return sp.all_see(a, j * BN, BN); };
        // ---- products ----
        const int slot = warp - C::MMA_WARP;
        const bool live = u.rows(a) > slot * kTileRows && u.rq.seq >= 0;
        const uint32_t id_s = idesc_f16(!Q8, false, BN), id_o = idesc_f16(!Q8, true, D);
        const uint32_t q_addr = smem_addr(smem) + slot * C::Q_BYTES, k_addr = smem_addr(smem + C::OFF_K), v_addr = smem_addr(smem + C::OFF_V);
        const uint32_t cols = tmem + (uint32_t)(slot * C::SLOT_COLS);
        // A group is P V of a tile and S of the one NSB after it, which goes over that P: the tensor pipe runs them in order. Each
        // group is waited for as a whole, and the slots' groups take turns: with both threads issuing as they could, the pipe
        // took their products alternately, so that both slots had their S at the same time and then waited for the
        // exponential unit together (5800 cycles a tile).
        auto ready_s = [&](int i) { return warp_wait(smem_addr(&sh.full_k[(it + i) % NS]), ((it + i) / NS) & 1, abort); };
        auto issue_s = [&](int i) {
            const int at = it + i, st = at % NS;
            if (!live) {
                mbar_arrive(smem_addr(&sh.s_full[slot][at % C::NSF]));
                return;
            }
            const uint32_t s_at = cols + (uint32_t)(C::S_COL + (at % NSB) * BN);
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
            mma_commit(smem_addr(&sh.s_full[slot][at % C::NSF]));
        };
        auto ready_pv = [&](int i) {
            const int at = it + i, st = at % NS;
            if (!warp_wait(smem_addr(&sh.full_v[st]), (at / NS) & 1, abort)) return false;
            if (!Q8 && !unit_sees(u.t0 + i)) {
                if (!warp_wait(smem_addr(&sh.v_clean[st]), (clean_phase >> st) & 1u, abort)) return false;
                clean_phase ^= 1u << st;
            }
            return warp_wait(smem_addr(&sh.p_full[slot][at % NSB]), (at / NSB) & 1, abort);
        };
        auto issue_pv = [&](int i) {
            const int at = it + i, st = at % NS;
            if (!live) {
                mbar_arrive(smem_addr(&sh.v_free[st]));
                return;
            }
            const uint32_t p_at = cols + (uint32_t)(C::S_COL + (at % NSB) * BN);
            const uint64_t vb = sdesc(v_addr + st * C::KV_BYTES, 1024, C::SBO, C::LAYOUT);
#pragma unroll
            for (int s4 = 0; s4 < BN / 64; ++s4) {
                uint32_t av[4];
                uint64_t bv[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int k = 4 * s4 + s;  // 16 keys
                    av[s] = p_at + (uint32_t)(32 * (k / 2) + 8 * (k % 2));  // (32 keys' P over their own scores)
                    bv[s] = vb + ((uint32_t)(k * 2 * C::SBO) >> 4);
                }
                mma_ts_x4<false>(cols + C::O_COL, av, bv, id_o, i > 0 || s4 > 0 ? 1u : 0u);
            }
            mma_commit(smem_addr(&sh.v_free[st]));
        };
        if (live) ok = ok && warp_wait(smem_addr(&sh.q_ready[slot]), live_units & 1, abort);
        for (int i = -NSB; ok && i < n; ++i) {
            const bool pv = i >= 0, next_s = i + NSB < n;
            if (RT == 1) {
                // (K may come from a stage whose V waits for this P V)
                if (pv) ok = ready_pv(i);
                tc_fence_after();
                if (ok && pv && elect_one()) issue_pv(i);
                __syncwarp();
                if (next_s) ok = ok && ready_s(i + NSB);
                tc_fence_after();
                if (ok && next_s && elect_one()) issue_s(i + NSB);
                __syncwarp();
                continue;
            }
            if (next_s) ok = ready_s(i + NSB);
            if (pv) ok = ok && ready_pv(i);
            // (the first slot's first turn is free)
            ok = ok && warp_wait(smem_addr(&sh.turn[slot]), (turns + (slot == 0 ? 1 : 0)) & 1, abort);
            ++turns;
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                if (pv) issue_pv(i);
                if (next_s) issue_s(i + NSB);
                mbar_arrive(smem_addr(&sh.turn[slot ^ 1]));
            }
            __syncwarp();
        }
        if (live && elect_one()) mma_commit(smem_addr(&sh.o_done[slot]));
        __syncwarp();
        if (!ok) *abort = 1;
        it += n;
        if (live) ++live_units;
    }
    // no product is left that uses the tensor memory
    if (elect_one()) mma_commit(smem_addr(&sh.drained[warp - C::MMA_WARP]));
    __syncwarp();
    mbar_wait_drain(smem_addr(&sh.drained[warp - C::MMA_WARP]), 0, kWait);
    return ok;
}

template <int D, bool Q8>
__device__ __forceinline__ bool softmax(const WindowArgs &a, uint8_t *smem, WShared &sh, Units<WCfg<D, Q8>::RT * kTileRows, WCfg<D, Q8>::BN> u, uint32_t tmem, int ctas, uint32_t total) {
    using C = WCfg<D, Q8>;
    constexpr int BN = C::BN, NS = C::NS, NSB = C::NSB, RT = C::RT, ROWS = RT * kTileRows;
    volatile int *abort = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // thread = row and 32 keys of a tile: two warps share 32 rows. A warp for all 64 keys waits for its own results (for the exponentials
    // alone 1.5 times what the special-function unit takes), and four to a scheduler fill one another's waits.
    constexpr int SHARE = C::SHARE, KEYS = BN / SHARE;
    const int slot = warp / (4 * SHARE), half = SHARE > 1 ? (warp >> 2) & 1 : 0, quarter = warp & 3, r = quarter * 32 + lane;
    [[maybe_unused]] const int id = 1 + slot * 4 + quarter;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(slot * C::SLOT_COLS);
    [[maybe_unused]] float *const x_mine = (float *)(smem + C::OFF_X) + (slot * 2 + half) * kTileRows + r, *const x_other = (float *)(smem + C::OFF_X) + (slot * 2 + 1 - half) * kTileRows + r;
    bool ok = true, fits = true;
    int it = 0, unit_no = 0;  // tiles and units of this CTA so far
    int live_units = 0;       // units that this slot had rows for
    int4 cut = make_int4(0, 0, 0, 0);  // the unit that this CTA begins and others end: row tile, KV head, last CTA
    // The unit's query rows of this warp: half of the 16-byte units of 32 rows, on their way, and there. A unit's rows are fetched as
    // soon as the products of the unit before are done, and the first scores run beside that unit's end.
    uint8_t *const q_rows = smem + slot * C::Q_BYTES + quarter * (C::Q_BYTES / 4);
    constexpr int QU = D / 8;
    auto q_fetch = [&](const auto &v) {
        const int row = v.row0 + slot * kTileRows + r, t = row_token(a, row);
        const long long q_at = ((long long)v.rq.src + t) * a.q_stride + (long long)(v.g * a.group + row - t * a.group) * D;
        const uint32_t have = __ballot_sync(0xffffffffu, row < v.rq.n * a.group);
#pragma unroll 2  // (more is slower: the end of a unit waits for its instructions)
        for (int k = 0; k < QU / SHARE; ++k) {
            const int i = (k * SHARE + half) * 32 + lane, rr = i / QU, uu = i % QU;
            const long long from = __shfl_sync(0xffffffffu, q_at, rr);
            const bool has = (have >> rr) & 1u;
            cp_async_16_or_zero(smem_addr(q_rows + bf16_off<D>(rr, 8 * uu)), has ? a.q + from + 8 * uu : a.q, has);
        }
    };
    auto q_there = [&] {
        cp_async_wait_all();
        if constexpr (Q8) {  // as f16, each lane what it fetched
#pragma unroll 2
            for (int k = 0; k < QU / SHARE; ++k) {
                const int i = (k * SHARE + half) * 32 + lane;
                uint4 *const at = (uint4 *)(q_rows + bf16_off<D>(i / QU, 8 * (i % QU)));
                const uint4 v = *at;
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float lo = __uint_as_float(w[e] << 16), hi = __uint_as_float(w[e] & 0xffff0000u);
                    fits = fits && fabsf(lo) <= 65504.0f && fabsf(hi) <= 65504.0f;
                    const __half2 h = __floats2half2_rn(lo, hi);
                    o[e] = *(const uint32_t *)&h;
                }
                *at = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&sh.q_ready[slot]));
    };
    auto has_rows = [&](const auto &v) { return v.rows(a) > slot * kTileRows && v.rq.seq >= 0; };
    const uint64_t scale2 = pair_of(a.scale_log2, a.scale_log2);
    bool more = u.next(a, warp == 0 && lane == 0);
    if (more && has_rows(u)) {
        q_fetch(u);
        q_there();
    }
    while (more) {
        const int n = u.t1 - u.t0;
        const Span sp = u.span(a);
        const int row = u.row0 + slot * kTileRows + r, t = row_token(a, row);
        const bool on = row < u.rq.n * a.group;
        const long long out_at = (((int64_t)u.rq.src + t) * a.q_heads + u.g * a.group + row - t * a.group) * D;
        if (!has_rows(u)) {
            // in step with the tiles all the same: a barrier's parity tells two phases apart, so nobody may fall behind
            for (int i = 0; i < n; ++i, ++it) {
                ok = ok && warp_wait(smem_addr(&sh.s_full[slot][it % C::NSF]), (it / C::NSF) & 1, abort);
                if (lane == 0) mbar_arrive(smem_addr(&sh.p_full[slot][it % NSB]));
            }
            if (!ok) *abort = 1;
            if (u.rq.seq < 0 && on && u.t0 == 0)  // a refused request's rows are 0
                for (int c = half * D / SHARE; c < (half + 1) * D / SHARE; c += 8) *(uint4 *)(a.out + out_at + c) = make_uint4(0, 0, 0, 0);
            ++unit_no;
            more = u.next(a, warp == 0 && lane == 0);
            if (more && has_rows(u)) {
                q_fetch(u);
                q_there();
            }
            continue;
        }
        const bool live = __any_sync(0xffffffffu, on);
        float m = -INFINITY;
        uint64_t l0 = 0, l1 = 0;  // the row's sum over this warp's keys
        const int p = u.rq.pos0 + t;
        for (int i = 0; i < n; ++i, ++it) {
            const int sb = it % NSB, key = (u.t0 + i) * BN + KEYS * half;
            ok = ok && warp_wait(smem_addr(&sh.s_full[slot][it % C::NSF]), (it / C::NSF) & 1, abort);
            if (!ok) *abort = 1;
            tc_fence_after();
            if (live) {
                const uint32_t s_col = lane_base + (uint32_t)(C::S_COL + sb * BN + KEYS * half);
                uint32_t s[KEYS / 32][32];
                if constexpr (KEYS == 64) tmem_load32x2(s_col, s_col + 32, s[0], s[1]);
                else tmem_load32(s_col, s[0]);
                if (!sp.all_see(a, key, KEYS)) {
#pragma unroll
                    for (int c = 0; c < KEYS / 32; ++c) {
                        const uint32_t bits = on ? seen_bits(a, sp, p, key + 32 * c) : 0u;
                        if (KEYS > 32 && __all_sync(0xffffffffu, bits == 0xffffffffu)) continue;
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!((bits >> k) & 1u)) s[c][k] = 0xff800000u;
                    }
                }
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < KEYS / 32; ++c)
#pragma unroll
                    for (int k = 0; k < 32; k += 2) tops[k / 2 % 4] = max3(tops[k / 2 % 4], __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
                const float top = max3(max3(tops[0], tops[1], tops[2]), tops[3], -INFINITY);
                const float mt = top == -INFINITY ? -INFINITY : top * a.scale_log2;
                bool any;
                if constexpr (SHARE > 1) any = pair_any(id, mt > m + C::LIMIT);
                else any = __any_sync(0xffffffffu, mt > m + C::LIMIT);
                if (any) {  // (a unit's first tile, hardly ever later)
                    float both = mt;
                    if constexpr (SHARE > 1) {
                        *x_mine = mt;
                        pair_sync(id);
                        both = fmaxf(mt, *x_other);
                    }
                    const bool up = both > m + C::LIMIT;
                    const float f = up ? ex2(m - both) : 1.0f;  // (0 for the first)
                    if (up) m = both;
                    l0 = fma_pair(l0, pair_of(f, f), 0);
                    l1 = fma_pair(l1, pair_of(f, f), 0);
                    if (i > 0) {
                        // O of the tiles before is complete when V of the last one is free
                        ok = ok && warp_wait(smem_addr(&sh.v_free[(it - 1) % NS]), ((it - 1) / NS) & 1, abort);
                        tc_fence_after();
#pragma unroll 1
                        for (int c0 = half * D / SHARE; c0 < (half + 1) * D / SHARE; c0 += 8) {
                            uint32_t o[8];
                            tmem_load8(lane_base + C::O_COL + c0, o);
#pragma unroll
                            for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            tmem_st8(lane_base + C::O_COL + c0, o);
                        }
                    }
                }
                const float neg = m == -INFINITY ? 0.0f : Q8 ? C::HEADROOM - m : -m;
                const uint64_t neg2 = pair_of(neg, neg);
#pragma unroll
                for (int c = 0; c < KEYS / 32; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float2 v = of_pair(fma_pair(pair_of(__uint_as_float(s[c][2 * k]), __uint_as_float(s[c][2 * k + 1])), scale2, neg2));
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
                    tmem_st16(s_col + 32 * c, w);
                }
                tmem_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&sh.p_full[slot][sb]));
        }
        ok = ok && warp_wait(smem_addr(&sh.o_done[slot]), live_units & 1, abort);
        ++live_units;
        if (!ok) *abort = 1;
        tc_fence_after();
        // the unit's end: the next one's query rows are fetched beside it
        const auto last = u;
        const bool whole = u.t0 == 0 && u.t1 == u.n_tiles;
        if (u.t0 == 0 && u.t1 < u.n_tiles) {  // cut, and this is the first of its CTAs: place x is CTA ((x + 1) G - 1) / T's
            const unsigned long long end = (unsigned long long)u.at + (uint32_t)(u.n_tiles + kUnitCost);
            cut = make_int4(u.b * a.row_tiles + u.rt, u.g, (int)((end * ctas - 1) / total), 1);
        }
        more = u.next(a, warp == 0 && lane == 0);
        const bool fetch = more && has_rows(u);
        if (fetch) q_fetch(u);
        if (live) {
            const float2 la = of_pair(l0), lb = of_pair(l1);
            float l = (la.x + la.y) + (lb.x + lb.y);
            if constexpr (SHARE > 1) {
                *x_mine = l;  // (the other warp has read the maximum: its P is in O)
                pair_sync(id);
                l = half ? *x_other + l : l + *x_other;
            }
            const long long part = (2ll * blockIdx.x + (last.t0 == 0 ? 1 : 0)) * ROWS + slot * kTileRows + r;
            if (!whole && on && half == 0) a.ws_ml[part] = make_float4(m, l, 0.0f, 0.0f);
            const float f = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const int ub = unit_no % kBadUnits, n_bad = Q8 ? 0 : min(kBadChunks, *(volatile int *)&((WBad *)(smem + C::OFF_BAD))->n[ub]);
            const uint32_t have = __ballot_sync(0xffffffffu, on);
#pragma unroll 1
            for (int c0 = half * D / SHARE; ok && c0 < (half + 1) * D / SHARE; c0 += 32) {
                uint32_t o[32];
                tmem_load32(lane_base + C::O_COL + c0, o);
                // rare: values that are not finite, for the rows that see them
#pragma unroll 1
                for (int i = 0; i < n_bad; ++i)
#pragma unroll 1
                    for (uint32_t bits = ((WBad *)(smem + C::OFF_BAD))->keys[ub][i]; bits; bits &= bits - 1) {
                        const int key = ((WBad *)(smem + C::OFF_BAD))->first[ub][i] + __ffs(bits) - 1, slot_k = sp.slot(key);
                        if (!on || !(seen_bits(a, sp, p, key) & 1u)) continue;
                        const int e = slot_k / a.pool.block_tokens, blk = lookup_block(a.pool, last.rq.seq, e);
                        if (blk < 0) continue;
                        const uint8_t *tile = a.pool.prefix + prefix_tile_index(a.pool, a.layer, blk, 1, last.g) * a.pool.tile_bytes;
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            const float y = bf16_bits_to_f32(*(const uint16_t *)(tile + bf16_off<D>(slot_k - e * a.pool.block_tokens, c0 + c)));
                            if (!isfinite(y)) o[c] = __float_as_uint(__uint_as_float(o[c]) + y);
                        }
                    }
                // (a row without a key: its P were 0, and so are its columns, as the values that some rows do not see are finite)
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float2 y = of_pair(fma_pair(pair_of(__uint_as_float(o[k]), __uint_as_float(o[k + 1])), pair_of(f, f), 0));
                    o[k] = __float_as_uint(y.x);
                    o[k + 1] = __float_as_uint(y.y);
                }
                if (!whole) {
                    if (on)
#pragma unroll
                        for (int k = 0; k < 8; ++k) *(uint4 *)(a.ws_o + part * D + c0 + 4 * k) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                } else {
                    uint4 x[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = pack_bf16(__uint_as_float(o[8 * k + 2 * e]), __uint_as_float(o[8 * k + 2 * e + 1]));
                        x[k] = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                    transpose4(x, lane);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int i = (lane & ~3) + k;
                        const long long to = __shfl_sync(0xffffffffu, out_at, i);
                        if ((have >> i) & 1u) *(uint4 *)(a.out + to + c0 + 8 * (lane & 3)) = x[k];
                    }
                }
                if (fetch && c0 == half * D / SHARE) q_there();
            }
        }
        if (fetch && !(live && ok)) q_there();
        tc_fence_before();
        ++unit_no;
    }
    if (a.split == kCutUnits && threadIdx.x == 0) a.cuts[blockIdx.x] = cut;
    if (!__all_sync(0xffffffffu, fits) && lane == 0) report_error(a.pool.status, DEV_ERR_F16_RANGE, blockIdx.x, warp, 15);
    return ok;
}

template <int D, bool Q8>
__global__ void __launch_bounds__(WCfg<D, Q8>::THREADS, 1) window_tile_kernel(const WindowArgs a) {
    using C = WCfg<D, Q8>;
    constexpr int NS = C::NS, NSB = C::NSB, RT = C::RT;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    WShared &sh = *(WShared *)(smem + C::OFF_SH);
    static_assert(2 * C::CONV_WARPS <= 8 && sizeof(WShared) <= 2048 && sizeof(WBad) <= 8192, "barrier block");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = a.pool.kv_heads;

    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(smem_addr(&sh.full_k[i]), Q8 ? C::CONV_WARPS : 1);
            mbar_init(smem_addr(&sh.full_v[i]), Q8 ? C::CONV_WARPS : 1);
            mbar_init(smem_addr(&sh.v_free[i]), Q8 ? RT : RT + C::SCRUB_WARPS);
            mbar_init(smem_addr(&sh.v_clean[i]), C::SCRUB_WARPS);
        }
        for (int k = 0; k < RT; ++k) {
            for (int i = 0; i < C::NSF; ++i) mbar_init(smem_addr(&sh.s_full[k][i]), 1);
            for (int i = 0; i < NSB; ++i) mbar_init(smem_addr(&sh.p_full[k][i]), 4 * C::SHARE);
            mbar_init(smem_addr(&sh.q_ready[k]), 4 * C::SHARE);
            mbar_init(smem_addr(&sh.o_done[k]), 1);
            mbar_init(smem_addr(&sh.drained[k]), 1);
            mbar_init(smem_addr(&sh.turn[k]), 1);
        }
        for (int i = 0; Q8 && i < 2 * C::NR; ++i) {
            mbar_init(smem_addr(&sh.raw_full[i / C::NR][i % C::NR]), 1);
            mbar_init(smem_addr(&sh.raw_empty[i / C::NR][i % C::NR]), C::CONV_WARPS);
        }
        sh.abort = 0;
        if constexpr (!Q8)
            for (int i = 0; i < kBadUnits; ++i) ((WBad *)(smem + C::OFF_BAD))->n[i] = 0;
        mbar_init_fence();
    }
    grid_wait();
    // (tensor memory between the two launch points: ekv_tree_tile.cu says why)
    if (warp == C::MMA_WARP) tmem_alloc(smem_addr(&sh.tmem), C::COLS);
    tc_fence_before();
    using U = Units<RT * kTileRows, C::BN>;
    RangeStart start{};
    if (a.split) {
        // a head's places of each request, a warp per request, in shared memory that nothing else uses yet
        uint32_t *const places = (uint32_t *)smem;
        constexpr int WARPS = C::THREADS / 32;
        for (int b = warp; b < a.n_batch; b += WARPS) {
            const WinReq rq = load_win_req(a, b, blockIdx.x == 0 && lane == 0);
            uint32_t sum = 0;
            for (int rt = lane; rt < a.row_tiles; rt += 32) sum += U::cost_of(a, rq, rt);
            sum = __reduce_add_sync(0xffffffffu, sum);
            if (lane == 0) places[b] = sum;
        }
        __syncthreads();
        const Range rg = find_range<C::THREADS>(
            a.n_batch, hk, sh.range, [&](int i) { return Req{0, (int)places[i], 0}; }, [](const Req &r) { return r.n_prefix; });
        start.x = rg.lo;
        start.hi = rg.hi;
        start.total = rg.total;
        start.ctas = rg.ctas;
        start.b = rg.b;
        if (warp == 0 && rg.lo < rg.hi) {
            // the head, and its row tile: 32 row tiles' places at a time
            const uint32_t head = places[rg.b];
            start.g = (int)((rg.lo - rg.base) / head);
            start.at = rg.base + start.g * head;
            const WinReq rq = load_win_req(a, rg.b, false);
            for (int rt0 = 0;; rt0 += 32) {
                const uint32_t cost = U::cost_of(a, rq, rt0 + lane);
                uint32_t incl = cost;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += v;
                }
                const uint32_t here = __ballot_sync(0xffffffffu, rg.lo < start.at + incl);
                if (here || rt0 + 32 >= a.row_tiles) {
                    const int l = here ? __ffs(here) - 1 : 31;
                    start.rt = rt0 + l;
                    start.at += __shfl_sync(0xffffffffu, incl - cost, l);
                    break;
                }
                start.at += __shfl_sync(0xffffffffu, incl, 31);
            }
            if (lane == 0) sh.start = start;
        }
        if (Q8 && threadIdx.x == 0 && rg.lo >= rg.hi) sh.start = start;  // (for seen_scales_fit)
        __syncthreads();
        if (rg.lo < rg.hi) start = sh.start;
        __syncthreads();  // (query rows go where the places are)
    } else {
        if (Q8 && threadIdx.x == 0) sh.start = start;
        __syncthreads();
    }
    tc_fence_after();
    const uint32_t tmem = sh.tmem;  // (there is a barrier in either branch)
    grid_launch_next();

    const U u(start);
    bool ok = true;
    if (warp < C::ROW_WARPS) {
        if constexpr (C::SPLIT_REGS) warpgroup_reg_alloc<C::ROW_REGS>();
        ok = softmax<D, Q8>(a, smem, sh, u, tmem, start.ctas, start.total);
    } else {
        if constexpr (C::SPLIT_REGS) warpgroup_reg_dealloc<C::OTHER_REGS>();
        if (warp < C::FEED_WARP) {
            ok = products<D, Q8>(a, smem, sh, u, tmem);
        } else if constexpr (Q8) {
            if (warp < C::CONV_WARP) ok = feed<D, true>(a, smem, sh, u);
            else if (warp < C::WARPS) ok = convert<D, true>(a, smem, sh, u);
        } else {
            if (warp < C::SCRUB_WARP) ok = feed<D, false>(a, smem, sh, u);
            else if (warp < C::WARPS) ok = look_at_values<D, false>(a, smem, sh, u);
        }
    }
    if (!ok && lane == 0) report_error(a.pool.status, DEV_ERR_TIMEOUT, blockIdx.x, warp, 15);
    __syncthreads();
    if (warp == C::MMA_WARP) tmem_dealloc(tmem, C::COLS);
    if constexpr (Q8)
        if (warp == 0 && __any_sync(0xffffffffu, lane < 2 * C::CONV_WARPS && sh.unfit[lane]) && !seen_scales_fit<D>(a, U(sh.start), C::BN, lane) && lane == 0)
            report_error(a.pool.status, DEV_ERR_F16_RANGE, blockIdx.x, 0, 15);
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
int window_tile_keys() { return 64; }

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
