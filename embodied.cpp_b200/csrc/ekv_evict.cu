// ekv_evict.cu -- eviction from the paged cache by accumulated attention weight.
//
// Every (layer, request, KV head) keeps `keep` of its rows: the first tokens, the most recent ones, and the
// heaviest others (ties to the lower slot). Survivors below `keep` stay where they are; the i-th free slot
// takes the i-th survivor at or above `keep`. So the bytes moved go with the rows that left, not with the
// rows that stay: a cache that gave up 100 of 1100 rows moves at most 100. Sources and destinations are
// disjoint, so rows move in any order.
//   evict_select_kernel  one CTA per (layer, request, KV head): the keep-th largest key by radix selection on
//                        its bits, one bit per slot for the choice, then a slot for each survivor
//   evict_move_kernel    a warp per 32 slots moves the K and V rows of those that changed (the CTA that chose them,
//                        where they are few)
#include <algorithm>

#include "ekv_decode.cuh"
#include "ekv_internal.h"

namespace ekv {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;  // 11 bits of the key at a time: 11, 11, 10
constexpr int kMoveWarps = 8;
constexpr int64_t kMoveHere = 256 * 1024;  // bytes that one CTA moves itself

// Larger is kept first. Protected rows are above every weight, NaN is below.
__device__ __forceinline__ uint32_t evict_key(float w, bool safe) {
    if (safe) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);  // -0 counts as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int kCopies = 4;   // histograms, by lane: weights share few exponents, so lanes meet in few bins
constexpr int kList = 12288; // survivors listed in shared memory; where more move, each free slot searches for its own
constexpr int kInRegs = 16;  // keys a thread keeps (16384 slots); longer rows are read again by each pass

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
    uint32_t w = sums[lane];
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
__device__ __forceinline__ void move_rows(const EvictArgs &a, int lbh, int slot0, int from, MoveShared &ms) {
    const PoolView &p = a.pool;
    const int h = lbh % p.kv_heads, lb = lbh / p.kv_heads, b = lb % a.n_batch, layer = a.layer0 + lb / a.n_batch;
    const int lane = threadIdx.x & 31, slot = slot0 + lane;
    const int seq = a.seq_ids[b];
    bool move = slot < a.keep && from >= 0 && from != slot;
    int bs = -1, bd = -1;
    if (move) {
        bs = lookup_block(p, seq, from / p.block_tokens);
        bd = lookup_block(p, seq, slot / p.block_tokens);
        move = bs >= 0 && bd >= 0;
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
    const int g = q8 ? D / 32 : 0;
    for (int i = lane; i < n * 2 * g; i += 32) {
        const int m = i / (2 * g);
        int u = i - m * 2 * g;
        const int64_t base = (u >= g ? kv_bytes : 0) + (int64_t)p.block_tokens * D;
        if (u >= g) u -= g;
        const int rs = ms.rows[m] >> 16, rd = ms.rows[m] & 0xffff;
        *(uint16_t *)(ms.dst[m] + base + (rd * g + u) * 2) = *(const uint16_t *)(ms.src[m] + base + (rs * g + u) * 2);
    }
    __syncwarp();
}

__global__ void __launch_bounds__(kSelThreads, 1) evict_select_kernel(const EvictArgs a) {
    extern __shared__ uint32_t s_mem[];
    __shared__ __align__(16) SelShared sh;
    static_assert(sizeof(sh.hist) >= sizeof(MoveShared) * kSelThreads / 32, "the moves' tables fit the histograms");
    int turn = 0;
    decode::grid_wait();
    decode::grid_launch_next();
    const int hk = a.pool.kv_heads;
    const int lbh = blockIdx.x, b = (lbh / hk) % a.n_batch;
    const int tid = threadIdx.x, lane = tid & 31;
    const int seq = a.seq_ids[b];
    int n = 0;
    if (seq < 0 || seq >= a.pool.max_seqs) {
        if (tid == 0) report_error(a.pool.status, DEV_ERR_BAD_SEQ, b, seq, 10);
    } else {
        n = a.pool.seq_lens[seq];
        if (n > a.weight_stride || n > a.max_len) {
            if (tid == 0) report_error(a.pool.status, DEV_ERR_BAD_POS, seq, n, 10);
            n = 0;
        }
    }
    const float *w = a.weights + (int64_t)lbh * a.weight_stride;
    const int32_t *pos = a.positions ? a.positions + (int64_t)lbh * a.weight_stride : nullptr;
    int32_t *kept = a.kept + (int64_t)lbh * a.keep;
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
    const bool in_regs = n <= kInRegs * kSelThreads;
    uint32_t keys[kInRegs];
    if (in_regs) {
#pragma unroll
        for (int j = 0; j < kInRegs; ++j) {
            const int i = tid + j * kSelThreads;
            keys[j] = i < n ? key_of(i) : 0u;
        }
    }
    // f(slot, key) for this thread's slots tid, tid + 1024, ...
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
#pragma unroll 1
    for (int pass = 0; pass < 3 && !all; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digits = pass == 2 ? 1024u : 2048u;
        for (int i = tid; i < kCopies * kBins; i += kSelThreads) (&sh.hist[0][0])[i] = 0;
        __syncthreads();
        each([&](int i, uint32_t k) {
            if (i < n && (k & mask) == prefix) atomicAdd(&sh.hist[lane % kCopies][(k >> shift) & (digits - 1)], 1u);
        });
        __syncthreads();
        // digits from the top: thread t holds digits 2 (1023 - t) + 1 and 2 (1023 - t)
        const int d = 2 * (kSelThreads - 1 - tid);
        uint32_t hi = 0, lo = 0;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
            const uint2 h = *(const uint2 *)&sh.hist[c][d];
            lo += h.x;
            hi += h.y;
        }
        uint32_t total;
        const uint32_t before = block_scan(hi + lo, sh, turn, total);
        if (before < need && need <= before + hi) {
            sh.digit = d + 1;
            sh.above = before;
            sh.count = hi;
        } else if (before + hi < need && need <= before + hi + lo) {
            sh.digit = d;
            sh.above = before + hi;
            sh.count = lo;
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
    each([&](int i, uint32_t k) {
        const uint32_t gt = __ballot_sync(0xffffffffu, i < n && (k & mask) > prefix);
        const uint32_t eq = __ballot_sync(0xffffffffu, i < n && (k & mask) == prefix);
        const int wd = i >> 5;
        if (lane == 0 && wd < words) {
            sel[wd] = gt;
            cnt[wd] = eq;
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
        for (int i = (a.keep & ~31) + tid; i < 32 * words; i += kSelThreads) {
            const int wd = i >> 5;
            const uint32_t bits = tail_bits(wd);
            if ((bits >> lane) & 1u) list[(wd == first_tail ? 0u : cnt[wd]) + __popc(bits & ((1u << lane) - 1u))] = i;
        }
        __syncthreads();
    }
    MoveShared *ms = (MoveShared *)&sh.hist[0][0];  // (the histograms are done with)
    for (int i0 = 0; i0 < a.keep; i0 += kSelThreads) {
        const int i = i0 + tid;
        const bool in = i < a.keep;
        const uint32_t chosen = in ? sel[i >> 5] : 0xffffffffu;
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
        if (in) {
            kept[i] = from;
            const float wi = w[from];
            const int32_t pi = pos ? pos[from] : from;
            if (w_out) w_out[i] = wi;
            if (p_out) p_out[i] = pi;
        }
        if (a.move_here) move_rows(a, lbh, i0 + (tid & ~31), in ? from : -1, ms[tid >> 5]);
    }
}

__global__ void __launch_bounds__(kMoveWarps * 32) evict_move_kernel(const EvictArgs a, int chunks) {
    __shared__ MoveShared ms[kMoveWarps];
    decode::grid_wait();
    const int lbh = blockIdx.x / chunks, warp = threadIdx.x >> 5;
    const int slot0 = ((blockIdx.x - lbh * chunks) * kMoveWarps + warp) * 32, slot = slot0 + (threadIdx.x & 31);
    move_rows(a, lbh, slot0, slot < a.keep ? a.kept[(int64_t)lbh * a.keep + slot] : -1, ms[warp]);
}

}  // namespace

int launch_evict(EvictArgs a, int max_live, cudaStream_t s) {
    const int64_t n = (int64_t)a.n_layers * a.n_batch * a.pool.kv_heads;
    const int chunks = (a.keep + kMoveWarps * 32 - 1) / (kMoveWarps * 32);
    if (n * chunks > INT32_MAX) return EKV_ERR_INVALID_ARG;
    a.max_words = (a.max_len + 31) / 32 + 1;
    // At most max_live - keep rows of each (layer, request, KV head) move: few are moved by the CTA that chose them, which
    // saves a launch and its tail; more are spread over the GPU. 18 x 100 rows of 544 bytes: 12.6 us with a second launch,
    // 9.6 without.
    const int64_t most = (int64_t)std::max(0, max_live - a.keep) * 2 * a.pool.tile_bytes / a.pool.block_tokens;
    a.move_here = most <= kMoveHere;
    const size_t smem = ((size_t)a.max_words * 2 + kList) * sizeof(uint32_t);
    static std::atomic<uint64_t> smem_done{0};
    if (const int rc = decode::allow_smem(evict_select_kernel, ((EKV_MAX_EVICT_TOKENS / 32 + 1) * 2 + kList) * (int)sizeof(uint32_t), smem_done))
        return rc;
    if (const int rc = decode::launch_after(evict_select_kernel, (unsigned)n, kSelThreads, smem, s, a)) return rc;
    if (a.move_here) return EKV_OK;
    return decode::launch_after(evict_move_kernel, (unsigned)(n * chunks), kMoveWarps * 32, 0, s, a, chunks);
}

}  // namespace ekv
