// ekv_evict.cu -- eviction from the paged cache by accumulated attention weight.
//
// Every (layer, request, KV head) keeps `keep` of its rows: the first tokens, the most recent ones, and the
// heaviest others (ties to the lower slot). Survivors below `keep` stay where they are; the i-th free slot
// takes the i-th survivor at or above `keep`. So the bytes moved go with the rows that left, not with the
// rows that stay: a cache that gave up 100 of 1100 rows moves at most 100. Sources and destinations are
// disjoint, so rows move in any order.
//   evict_select_kernel  one CTA per (layer, request, KV head): the keep-th largest key by radix selection on
//                        its bits, one bit per slot for the choice, then a slot for each survivor
//   evict_move_kernel    a warp per 32 slots moves the K and V rows of those that changed
// Bounds and figures: the move is bound by DRAM (64 rows of 16384 slots cut to 4096, head_dim 128 bf16: 38 us where the
// bytes alone would take 31), the selection by its instructions and barriers, not by bytes (14 us for those 64 rows,
// whose weights would take 0.6). Moving the rows in the CTA that chose them saved the second
// launch on the host but left a third of the SMs to move everything: 14.0 us against 13.3 for 18 rows of 1100 slots.
#include <algorithm>

#include "ekv_decode.cuh"
#include "ekv_internal.h"

namespace ekv {
namespace {

// Threads of a selection: 512 for rows of up to kFewSlots slots, whose barriers cost more than their keys (18 rows of
// 1100 slots, the move included: 11.7 us, against 12.8 with 256 threads and 12.6 with 1024, all with 8 moving warps), else 1024.
constexpr int kFewThreads = 512, kManyThreads = 1024, kFewSlots = 4096;
constexpr int kBins = 2048;  // 11 bits of the key at a time: 11, 11, 10
// Warps of a moving CTA: few, so that the last wave of CTAs is a short one (64 rows of 16384 slots cut to 4096, the
// selection included: 56.0 us with 8 warps, 54.1 with 2).
constexpr int kMoveWarps = 2;

// Larger is kept first. Protected rows are above every weight, NaN is below.
__device__ __forceinline__ uint32_t evict_key(float w, bool safe) {
    const uint32_t b = __float_as_uint(w + 0.0f);  // -0 counts as 0
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return safe ? 0xffffffffu : w != w ? 0u : k;
}

constexpr int kCopies = 4;   // histograms, by lane: weights share few exponents, so lanes meet in few bins
constexpr int kList = 12288; // survivors listed in shared memory; where more move, each free slot searches for its own
// Keys a thread keeps (16384 slots); longer rows are read again by each pass: 64 rows cut to 4096 take 54 us from 16000 slots,
// 63 from 17000, 130 from 60000, 16 rows 560 from 400000.
constexpr int kInRegs = 16;

struct SelShared {
    uint32_t hist[kCopies][kBins];
    uint32_t warp_sum[2][32];
    uint32_t digit, above, count;
};

// Block-wide exclusive scan of one value per thread; the total in `total`. One barrier: consecutive scans
// alternate between two buffers (`turn`).
__device__ __forceinline__ uint32_t block_scan(uint32_t v, SelShared &sh, int &turn, uint32_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t *sums = sh.warp_sum[turn];
    turn ^= 1;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    uint32_t w = lane < (int)blockDim.x / 32 ? sums[lane] : 0u;
    const uint32_t mine = __shfl_sync(0xffffffffu, w, warp);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += u;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    return s - v + __shfl_sync(0xffffffffu, w, warp) - mine;
}

// A warp's 32 slots of (layer, request, KV head) lbh: those whose row comes from elsewhere get it, K and V.
struct MoveShared {
    const uint8_t *src[32];
    uint8_t *dst[32];
    int rows[32];  // row inside the source block << 16 | inside the destination block
};
template <class From>
__device__ __forceinline__ void move_rows(const EvictArgs &a, int lbh, int slot0, From from_of, MoveShared &ms) {
    const PoolView &p = a.pool;
    const int h = lbh % p.kv_heads, lb = lbh / p.kv_heads, b = lb % a.n_batch, layer = a.layer0 + lb / a.n_batch;
    const int lane = threadIdx.x & 31, slot = slot0 + lane;
    // What the selection does not write is read while it still runs: it let this grid start after its own wait.
    const int seq = a.seq_ids[b];
    const bool real = slot < a.keep && seq >= 0 && seq < p.max_seqs && slot < p.seq_lens[seq];
    const int bd = real ? lookup_block(p, seq, slot / p.block_tokens) : -1;
    decode::grid_wait();
    const int from = bd >= 0 ? from_of(slot) : -1;
    bool move = from >= 0 && from != slot;
    int bs = -1;
    if (move) {
        bs = lookup_block(p, seq, from / p.block_tokens);
        move = bs >= 0;
    }
    const uint32_t moving = __ballot_sync(0xffffffffu, move);
    if (!moving) return;
    const int n = __popc(moving);
    if (move) {
        const int i = __popc(moving & ((1u << lane) - 1u));
        ms.src[i] = p.prefix + prefix_tile_index(p, layer, bs, 0, h) * p.tile_bytes;
        ms.dst[i] = p.prefix + prefix_tile_index(p, layer, bd, 0, h) * p.tile_bytes;
        ms.rows[i] = from % p.block_tokens << 16 | slot % p.block_tokens;
    }
    __syncwarp();
    const int D = p.head_dim;
    const int64_t kv_bytes = (int64_t)p.kv_heads * p.tile_bytes;
    const bool q8 = p.dtype == EKV_DTYPE_Q8_0;
    const int per = q8 ? D / 16 : D / 8, units = 2 * per;  // 16-byte units of a row, K then V
    // Q8_0 scales, 2 bytes each: the first of them on their way before the rows
    const int g = q8 ? D / 32 : 0, n_scales = n * 2 * g;
    constexpr int EARLY = 4;
    auto scale_at = [&](int i, bool to) -> uint16_t * {
        const int m = i / (2 * g);
        int u = i - m * 2 * g;
        const int64_t base = (u >= g ? kv_bytes : 0) + (int64_t)p.block_tokens * D;
        if (u >= g) u -= g;
        return to ? (uint16_t *)(ms.dst[m] + base + ((ms.rows[m] & 0xffff) * g + u) * 2)
                  : (uint16_t *)(ms.src[m] + base + ((ms.rows[m] >> 16) * g + u) * 2);
    };
    uint16_t early[EARLY];
#pragma unroll
    for (int j = 0; j < EARLY; ++j)
        if (lane + 32 * j < n_scales) early[j] = *scale_at(lane + 32 * j, false);
    // A lane keeps one unit of the row; where a row has at most 16 units, several rows are taken at a time.
    const int wlog = decode::log2_of(p.swz_bytes);
    const int at_once = units <= 16 ? 32 / units : 1, sub = units <= 16 ? lane / units : 0;
    constexpr int UNROLL = 8;
    for (int u0 = units <= 16 ? lane - sub * units : lane; u0 < units; u0 += 32) {
        if (sub >= at_once) break;
        const int u = u0 >= per ? u0 - per : u0;
        const int64_t kv = u0 >= per ? kv_bytes : 0;
        for (int m0 = sub; m0 < n; m0 += at_once * UNROLL) {
            uint4 v[UNROLL];
#pragma unroll
            for (int j = 0; j < UNROLL; ++j) {
                const int m = m0 + j * at_once;
                if (m >= n) continue;
                const int rs = ms.rows[m] >> 16;
                v[j] = *(const uint4 *)(ms.src[m] + kv + (q8 ? q8_qs_off(rs, 16 * u, D) : decode::bf16_off_any(rs, 8 * u, D, wlog)));
            }
#pragma unroll
            for (int j = 0; j < UNROLL; ++j) {
                const int m = m0 + j * at_once;
                if (m >= n) continue;
                const int rd = ms.rows[m] & 0xffff;
                *(uint4 *)(ms.dst[m] + kv + (q8 ? q8_qs_off(rd, 16 * u, D) : decode::bf16_off_any(rd, 8 * u, D, wlog))) = v[j];
            }
        }
    }
#pragma unroll
    for (int j = 0; j < EARLY; ++j)
        if (lane + 32 * j < n_scales) *scale_at(lane + 32 * j, true) = early[j];
    for (int i = lane + 32 * EARLY; i < n_scales; i += 32) *scale_at(i, true) = *scale_at(i, false);
    __syncwarp();
}

template <int kSelThreads>
__global__ void __launch_bounds__(kSelThreads, 1) evict_select_kernel(const EvictArgs a) {
    extern __shared__ uint32_t s_mem[];
    __shared__ __align__(16) SelShared sh;
    int turn = 0;
    decode::grid_wait();
    decode::grid_launch_next();
    const int hk = a.pool.kv_heads;
    const int lbh = blockIdx.x, b = (lbh / hk) % a.n_batch;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seq = a.seq_ids[b];
    const float *w = a.weights + (int64_t)lbh * a.weight_stride;
    const int32_t *pos = a.positions ? a.positions + (int64_t)lbh * a.weight_stride : nullptr;
    // The row is asked for before its length is known: the sequence's id and length are two reads one after the other.
    // All of a thread's loads come first: with the test of each key between them a row of 16384 took 10 us to read.
    const int ahead = min(a.row_hint, kInRegs * kSelThreads);
    uint32_t keys[kInRegs], ages[kInRegs];
#pragma unroll
    for (int j = 0; j < kInRegs; ++j) {
        const int i = tid + j * kSelThreads;
        keys[j] = i < ahead ? __float_as_uint(__ldg(w + i)) : 0u;
    }
#pragma unroll
    for (int j = 0; j < kInRegs; ++j) {
        const int i = tid + j * kSelThreads;
        ages[j] = pos && i < ahead ? (uint32_t)__ldg(pos + i) : (uint32_t)i;
    }
    int n = -1;
    if (seq < 0 || seq >= a.pool.max_seqs) {
        if (tid == 0) report_error(a.pool.status, DEV_ERR_BAD_SEQ, b, seq, 10);
    } else {
        n = a.pool.seq_lens[seq];
        if (n > a.weight_stride || n > a.max_len) {
            if (tid == 0) report_error(a.pool.status, DEV_ERR_BAD_POS, seq, n, 10);
            n = -1;
        }
    }
    int32_t *kept = a.kept + (int64_t)lbh * a.keep;
    if (n < 0) {  // reported: no row moves, and weights and positions, which may be the call's own inputs, stay
        for (int i = tid; i < a.keep; i += kSelThreads) kept[i] = -1;
        return;
    }
    float *w_out = a.weights_out ? a.weights_out + (int64_t)lbh * a.out_stride : nullptr;
    int32_t *p_out = a.positions_out ? a.positions_out + (int64_t)lbh * a.out_stride : nullptr;
    const int recent_from = (a.seen ? a.seen[b] : n) - a.recent;
    auto key_of = [&](int i) {
        const int age = pos ? pos[i] : i;
        return evict_key(w[i], age < a.first || age >= recent_from);
    };

    if (n <= a.keep) {  // everything stays
        for (int i = tid; i < a.keep; i += kSelThreads) {
            const bool on = i < n;
            kept[i] = on ? i : -1;
            const float wi = on ? w[i] : 0.0f;
            const int32_t pi = on ? (pos ? pos[i] : i) : -1;
            if (w_out) w_out[i] = wi;
            if (p_out) p_out[i] = pi;
        }
        return;
    }

    // ---- the keep-th largest key, from its upper bits down ----
    const bool in_regs = n <= ahead;
#pragma unroll
    for (int j = 0; j < kInRegs; ++j) {
        const int age = (int)ages[j];
        keys[j] = evict_key(__uint_as_float(keys[j]), age < a.first || age >= recent_from);
    }
    // f(slot, key) for this thread's slots tid, tid + kSelThreads, ...
    auto each = [&](auto f) {
        if (in_regs) {
#pragma unroll
            for (int j = 0; j < kInRegs; ++j) {
                if (j * kSelThreads >= n) break;
                f(tid + j * kSelThreads, keys[j]);
            }
        } else {
#pragma unroll 4
            for (int i = tid; i - tid < n; i += kSelThreads) f(i, i < n ? key_of(i) : 0u);
        }
    };
    uint32_t prefix = 0, mask = 0;
    uint32_t need = (uint32_t)a.keep;  // how many of the keys that match `prefix` are kept
    bool all = false;                  // every key that matches is kept
    for (int i = tid; i < kCopies * kBins / 2; i += kSelThreads) ((uint2 *)&sh.hist[0][0])[i] = make_uint2(0, 0);
    __syncthreads();
#pragma unroll 1
    for (int pass = 0; pass < 3 && !all; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digits = pass == 2 ? 1024u : 2048u;
        each([&](int i, uint32_t k) {
            if (i < n && (k & mask) == prefix) atomicAdd(&sh.hist[lane % kCopies][(k >> shift) & (digits - 1)], 1u);
        });
        __syncthreads();
        // digits from the top: thread t holds the PER digits from PER (threads - 1 - t); cleared for the next pass
        constexpr int PER = kBins / kSelThreads;
        struct __align__(4 * PER) Digits {
            uint32_t n[PER];
        };
        const int d = PER * (kSelThreads - 1 - tid);
        uint32_t cnt[PER], sum = 0;
#pragma unroll
        for (int e = 0; e < PER; ++e) cnt[e] = 0;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
            Digits *h = (Digits *)&sh.hist[c][d];
            const Digits v = *h;
#pragma unroll
            for (int e = 0; e < PER; ++e) cnt[e] += v.n[e];
            *h = Digits{};
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) sum += cnt[e];
        // only the warp in which the count reaches `need` looks closer
        const uint32_t mine = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0) sh.warp_sum[0][warp] = mine;
        __syncthreads();
        const uint32_t above = __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_sum[0][lane] : 0u);  // (warp 0: none)
        if (above < need && need <= above + mine) {
            uint32_t s = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t u = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += u;
            }
            uint32_t before = above + s - sum;
#pragma unroll
            for (int e = PER - 1; e >= 0; --e) {
                if (before < need && need <= before + cnt[e]) {
                    sh.digit = d + e;
                    sh.above = before;
                    sh.count = cnt[e];
                }
                before += cnt[e];
            }
        }
        __syncthreads();
        prefix |= sh.digit << shift;
        mask |= (digits - 1) << shift;
        need -= sh.above;
        all = sh.count == need;
    }
    // kept: keys above `prefix` in the digits seen, and the first `need` equal to it there

    // ---- one bit per slot ----
    const int words = (n + 31) / 32;
    uint32_t *sel = s_mem, *cnt = s_mem + a.max_words;  // chosen slots; ties, then free slots or survivors before a word
    uint32_t *list = s_mem + 2 * a.max_words;           // [kList] survivors at or above keep
    if (all) {  // (the usual case: no tie at the last place)
        each([&](int i, uint32_t k) {
            const uint32_t in = __ballot_sync(0xffffffffu, i < n && (k & mask) >= prefix);
            if (lane == 0 && i < n) sel[i >> 5] = in;
        });
    } else {
        each([&](int i, uint32_t k) {
            const uint32_t gt = __ballot_sync(0xffffffffu, i < n && (k & mask) > prefix);
            const uint32_t eq = __ballot_sync(0xffffffffu, i < n && (k & mask) == prefix);
            if (lane == 0 && i < n) {
                sel[i >> 5] = gt;
                cnt[i >> 5] = eq;
            }
        });
        __syncthreads();
        uint32_t ties = 0;
        for (int w0 = 0; w0 < words; w0 += kSelThreads) {
            const int wd = w0 + tid;
            const uint32_t eq = wd < words ? cnt[wd] : 0u;
            uint32_t total;
            uint32_t rank = ties + block_scan(__popc(eq), sh, turn, total);
            if (eq && rank < need) {
                uint32_t take = need - rank, e = eq, got = 0;
                if (take >= (uint32_t)__popc(eq)) {
                    got = eq;
                } else {
                    for (; take; --take) {
                        got |= e & (0u - e);
                        e &= e - 1;
                    }
                }
                sel[wd] |= got;
            }
            ties += total;
        }
    }
    __syncthreads();
    // ---- survivors at or above keep before each word ----
    const int first_tail = a.keep >> 5;  // the word that holds slot keep
    auto tail_bits = [&](int wd) {
        return wd < first_tail ? 0u : wd == first_tail ? sel[wd] & ~((1u << (a.keep & 31)) - 1u) : sel[wd];
    };
    // (cnt of a word below holds the free slots before it)
    const uint32_t low_mask = (1u << (a.keep & 31)) - 1u;
    uint32_t tails = 0, holes = 0;
    for (int w0 = 0; w0 < words; w0 += kSelThreads) {
        const int wd = w0 + tid;
        const uint32_t free_bits = wd >= words || wd > first_tail ? 0u : wd < first_tail ? ~sel[wd] : ~sel[wd] & low_mask;
        const uint32_t tail = wd < words ? tail_bits(wd) : 0u;
        uint32_t total;
        // both counts in one scan: each is at most 2^15 a round
        const uint32_t before = block_scan(__popc(tail) << 16 | __popc(free_bits), sh, turn, total);
        if (wd < words) cnt[wd] = wd <= first_tail ? holes + (before & 0xffffu) : tails + (before >> 16);
        tails += total >> 16;
        holes += total & 0xffffu;
    }
    __syncthreads();
    // ---- the survivors in order, and a free slot below keep for each ----
    const bool listed = holes <= (uint32_t)kList;
    if (listed) {
        for (int i = 4 * first_tail + tid; i < 4 * words; i += kSelThreads) {  // eight slots each
            const int wd = i >> 2, lo = 8 * (i & 3);
            const uint32_t word = tail_bits(wd);
            uint32_t at = (wd == first_tail ? 0u : cnt[wd]) + __popc(word & ((1u << lo) - 1u));
            for (uint32_t bits = (word >> lo) & 0xffu; bits; bits &= bits - 1) list[at++] = 32 * wd + lo + __ffs(bits) - 1;
        }
        __syncthreads();
    }
    for (int i = tid; i < a.keep; i += kSelThreads) {
        const uint32_t chosen = sel[i >> 5];
        int from = i;
        if (!((chosen >> (i & 31)) & 1u)) {
            const uint32_t rank = cnt[i >> 5] + __popc(~chosen & ((1u << (i & 31)) - 1u));
            if (listed) {
                from = list[rank];
            } else {
                int lo = first_tail, hi = words - 1;  // the last word with at most `rank` survivors before it
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (cnt[mid] <= rank) lo = mid;
                    else hi = mid - 1;
                }
                uint32_t bits = tail_bits(lo);
                for (uint32_t k = rank - (lo == first_tail ? 0u : cnt[lo]); k; --k) bits &= bits - 1;
                from = 32 * lo + __ffs(bits) - 1;
            }
        }
        kept[i] = from;
        const float wi = w[from];
        const int32_t pi = pos ? pos[from] : from;
        if (w_out) w_out[i] = wi;
        if (p_out) p_out[i] = pi;
    }
}

__global__ void __launch_bounds__(kMoveWarps * 32) evict_move_kernel(const EvictArgs a, int chunks) {
    __shared__ MoveShared ms[kMoveWarps];
    const int lbh = blockIdx.x / chunks, warp = threadIdx.x >> 5;
    const int slot0 = ((blockIdx.x - lbh * chunks) * kMoveWarps + warp) * 32;
    move_rows(a, lbh, slot0, [&](int slot) { return a.kept[(int64_t)lbh * a.keep + slot]; }, ms[warp]);
}

}  // namespace

int launch_evict(EvictArgs a, int max_live, cudaStream_t s) {
    const int64_t n = (int64_t)a.n_layers * a.n_batch * a.pool.kv_heads;
    const int chunks = (a.keep + kMoveWarps * 32 - 1) / (kMoveWarps * 32);
    if (n * chunks > INT32_MAX) return EKV_ERR_INVALID_ARG;
    a.max_words = (a.max_len + 31) / 32 + 1;
    const size_t smem = ((size_t)a.max_words * 2 + kList) * sizeof(uint32_t);
    // The longest live sequence and the stride bound the rows of the call, which are known on the device: they pick the form
    // and how much of a row is read ahead, and any sequence is right with either. A longer sequence that is not of the call
    // counts only where the stride has room for it: 18 rows of 1100 slots 9.6 us, 10.8 with a stride of 20480 and such a
    // sequence beside them; 64 rows of 16000 slots 54 us either way.
    a.row_hint = (int)std::min<int64_t>(std::min(max_live, a.max_len), a.weight_stride);
    const bool few = a.row_hint <= kFewSlots;
    static std::atomic<uint64_t> few_done{0}, many_done{0};
    const int most_smem = ((EKV_MAX_EVICT_TOKENS / 32 + 1) * 2 + kList) * (int)sizeof(uint32_t);
    int rc = few ? decode::allow_smem(evict_select_kernel<kFewThreads>, most_smem, few_done)
                 : decode::allow_smem(evict_select_kernel<kManyThreads>, most_smem, many_done);
    if (!rc)
        rc = few ? decode::launch_after(evict_select_kernel<kFewThreads>, (unsigned)n, kFewThreads, smem, s, a)
                 : decode::launch_after(evict_select_kernel<kManyThreads>, (unsigned)n, kManyThreads, smem, s, a);
    if (rc) return rc;
    return decode::launch_after(evict_move_kernel, (unsigned)(n * chunks), kMoveWarps * 32, 0, s, a, chunks);
}

}  // namespace ekv
