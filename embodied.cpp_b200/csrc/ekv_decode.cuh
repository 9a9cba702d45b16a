// ekv_decode.cuh -- shared parts of the decoding kernels over the paged pool (draft-tree attention and
// key weights): work partition over ragged requests, the copy-engine feeder of 64-key tiles, and the
// warp-level matrix instructions with their shared-memory operand loads.
//
// These kernels have few query rows per cached key (one row per drafted token and query head of a KV
// head's group), so the bytes of the cache bound them, not the tensor pipe: 16 rows take
// 32 * head_dim multiply-adds per key of 4 * head_dim bytes. mma.sync with operands in registers keeps
// the whole row state (maximum, sum, output) in one warp and needs no tensor-memory round trip per tile.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "ekv_device.cuh"
#include "ekv_internal.h"
#include "ekv_sm100.cuh"

namespace ekv {
namespace decode {

// ---- launches ----
// The decoding calls are short and follow one another, so their kernels start while the one before them in the
// stream drains (programmatic launch): each waits for it with grid_wait() before it touches global memory.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... P, class... A>
int launch_clusters_after(int cluster, void (*k)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, const A &...args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3((unsigned)threads);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = cluster > 1 ? 2 : 1;
    if (cudaLaunchKernelEx(&c, k, P(args)...) != cudaSuccess) {
        cudaGetLastError();
        return EKV_ERR_CUDA;
    }
    note_launches(1);
    return EKV_OK;
}

template <class... P, class... A>
int launch_after(void (*k)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, const A &...args) {
    return launch_clusters_after(1, k, grid, threads, smem, s, args...);
}

// Dynamic shared memory above 48 KB, asked for once per kernel and device (`done`: the devices asked on).
template <class K>
int allow_smem(K k, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return EKV_ERR_CUDA;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return EKV_OK;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
        cudaGetLastError();
        return EKV_ERR_CUDA;
    }
    done.fetch_or(bit, std::memory_order_relaxed);
    return EKV_OK;
}

// Bounded wait of a whole warp: the same answer in every lane, so that what follows may be warp-wide.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort) {
    return __all_sync(0xffffffffu, sm100::mbar_wait(bar, parity, abort, kDefaultWaitBudget));
}

constexpr int kTile = 64;                       // keys per tile
constexpr long long kWait = kDefaultWaitBudget; // clock cycles a bounded wait gives up after

// ---- storage of a tile in shared memory ----
template <int D, bool Q8>
struct TileCfg {
    static constexpr int W = (D * 2) % 128 == 0 ? 128 : (D * 2) % 64 == 0 ? 64 : 32;  // swizzle chunk (bf16)
    static constexpr int G32 = D / 32;                                                // Q8_0 scale groups
    static constexpr int KV_BYTES = Q8 ? kTile * D + kTile * G32 * 2 : kTile * D * 2; // K or V of a tile
    static constexpr int SCALES = kTile * D;  // offset of the scales (Q8_0)
};

// Byte offset of (row, d) of a bf16 tile, compile-time head_dim.
template <int D>
__device__ __forceinline__ uint32_t bf16_off(int row, int d) {
    constexpr int W = TileCfg<D, false>::W;
    return tile_elem_off(row, d, D, W);
}

// The same with run-time head_dim, for kernels of any: 8 W bytes of 2 D / W chunks are 16 D bytes per 8 rows, and
// W = 2^w, so that no division is left.
__device__ __forceinline__ uint32_t bf16_off_any(int row, int d, int D, int w) {
    const int byte = 2 * d;
    return (uint32_t)((row >> 3) * 16 * D + ((byte >> w) << (w + 3))) +
           swz((uint32_t)(((row & 7) << w) + (byte & ((1 << w) - 1))), (1u << (w - 4)) - 1);
}
__device__ __forceinline__ int log2_of(int pow2) { return 31 - __clz(pow2); }

// ---- matrix instructions ----
// D[16x8] += A[16x16] * B[16x8], bf16 operands, f32 accumulators.
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
// The G f16 scales of one key's row, two to a word, and one of them.
template <int G>
__device__ __forceinline__ void load_scales(uint32_t addr, uint32_t (&s)[(G + 1) / 2]) {
    static_assert(G % 2 == 0, "whole words");
    if constexpr (G % 8 == 0) {
#pragma unroll
        for (int i = 0; i < G / 8; ++i) {
            const uint4 v = lds128(addr + 16 * i);
            s[4 * i] = v.x;
            s[4 * i + 1] = v.y;
            s[4 * i + 2] = v.z;
            s[4 * i + 3] = v.w;
        }
    } else if constexpr (G % 4 == 0) {
#pragma unroll
        for (int i = 0; i < G / 4; ++i) {
            const uint2 v = lds64(addr + 8 * i);
            s[2 * i] = v.x;
            s[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < G / 2; ++i) s[i] = lds32(addr + 4 * i);
    }
}
template <int N>
__device__ __forceinline__ float scale_of(const uint32_t (&s)[N], int g) {
    const __half2 h = *(const __half2 *)&s[g >> 1];
    return g & 1 ? __high2float(h) : __low2float(h);
}
// 16 bytes to another CTA's shared memory (address from mapa_shared).
__device__ __forceinline__ void stc128(uint32_t addr, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The same, or 16 zero bytes where `on` is false (the source is not read then).
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst, const void *src, bool on) {
    const int n = on ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *(const uint32_t *)&h;
}

// Pairs of f32 in one 64-bit register: one instruction for two products or sums.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 of_pair(uint64_t p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// Four int8 of a word to two bf16 pairs, exactly: with x = low7 - 128 * sign, the bf16 with upper byte
// 0x43 and lower byte low7 is 128 + low7, and the one with lower byte (x & 0x80) is 128 or 256; their
// difference is x.
__device__ __forceinline__ void int8x4_to_bf16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t m = w & 0x7f7f7f7fu, s = w & 0x80808080u;
    const uint32_t a0 = __byte_perm(m, 0x43434343u, 0x4140), a1 = __byte_perm(m, 0x43434343u, 0x4342);
    const uint32_t b0 = __byte_perm(s, 0x43434343u, 0x4140), b1 = __byte_perm(s, 0x43434343u, 0x4342);
    const __nv_bfloat162 r0 = __hsub2(*(const __nv_bfloat162 *)&a0, *(const __nv_bfloat162 *)&b0);
    const __nv_bfloat162 r1 = __hsub2(*(const __nv_bfloat162 *)&a1, *(const __nv_bfloat162 *)&b1);
    lo = *(const uint32_t *)&r0;
    hi = *(const uint32_t *)&r1;
}

// Score of q.k in the log2 domain: scale * q.k * log2(e), or cap * tanh(scale * q.k / cap) * log2(e). The full
// tanhf: through exp(2y) the quotient loses 2^-23 of the cap near 0, several times what an uncapped score loses.
struct ScoreFn {
    float scale_log2;  // scale * log2(e)
    float cap_log2;    // cap * log2(e), 0 = no cap
    float cap_in;      // scale / cap
    __device__ __forceinline__ float capped(float s) const { return cap_log2 * tanhf(s * cap_in); }
    // N scores in place, behind one branch
    template <int N>
    __device__ __forceinline__ void operator()(float (&s)[N]) const {
        if (cap_log2 == 0.0f) {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] *= scale_log2;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] = capped(s[i]);
        }
    }
};

// ---- requests and the work partition ----
// One request of the call: cached keys [0, n_prefix) and n_nodes drafted tokens.
struct Req {
    int seq, n_prefix, n_nodes;
};

__device__ __forceinline__ Req load_req(const TreeArgs &a, int b, bool report) {
    Req r;
    r.seq = a.seq_ids[b];
    r.n_prefix = 0;
    r.n_nodes = a.n_draft;
    if (a.n_nodes) r.n_nodes = min(max(a.n_nodes[b], 0), a.n_draft);
    if (r.seq < 0 || r.seq >= a.pool.max_seqs) {
        if (report) report_error(a.pool.status, DEV_ERR_BAD_SEQ, b, r.seq, 5);
        r.seq = 0;
        return r;
    }
    const int len = a.pool.seq_lens[r.seq];
    const int np = a.prefix_len ? a.prefix_len[b] : len;
    if (np < 0 || np > len) {
        if (report) report_error(a.pool.status, DEV_ERR_BAD_POS, b, np, len);
        return r;
    }
    r.n_prefix = np;
    return r;
}

// A flat order of all tiles of the call -- request, then unit (KV head, row tile), then tile -- is cut
// into G = min(gridDim.x, T) equal ranges, whatever the requests' lengths: CTA c < G takes
// [c T / G, (c + 1) T / G), at least one tile. The launchers see to it that T < 2^31.
struct Range {
    uint32_t total, lo, hi;  // T and this CTA's range
    int ctas;                // G
    int b;                   // request that holds tile lo
    uint32_t base;           // first tile of request b
    Req req;                 // request b
};

struct RangeScratch {
    uint32_t warp_sum[32];
    uint32_t base;
    int b;
    Req req;
};

// floor(total * c / g) for c <= g <= 2^16, in 32 bits.
__device__ __forceinline__ uint32_t range_lo(uint32_t total, uint32_t c, uint32_t g) {
    const uint32_t q = total / g, r = total - q * g;
    return c * q + c * r / g;
}

// floor(row / group) for the row of a unit: row * group < 2^32 (checked at the call), group_mul = ceil(2^32 / group).
__device__ __forceinline__ int row_token(const TreeArgs &a, int row) {
    return a.group == 1 ? row : (int)__umulhi((uint32_t)row, a.group_mul);
}

// All threads of the block (NT of them). request(b): request b; tiles(r): tiles of one unit of a request.
template <int NT, class Request, class Tiles>
__device__ __forceinline__ Range find_range(int n_batch, int units_per_req, RangeScratch &sh, Request request, Tiles tiles) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = NT / 32;
    // inclusive scan of one chunk of NT requests; returns this thread's inclusive sum and the chunk's total
    auto scan = [&](uint32_t v, uint32_t &chunk) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) sh.warp_sum[warp] = v;
        __syncthreads();
        uint32_t before = 0;
        chunk = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const uint32_t s = sh.warp_sum[w];
            if (w < warp) before += s;
            chunk += s;
        }
        return v + before;
    };
    Range r;
    r.total = 0;
    Req mine{};
    if (tid < n_batch) mine = request(tid);
    const uint32_t v0 = tid < n_batch ? (uint32_t)(tiles(mine) * units_per_req) : 0u;
    uint32_t incl0 = 0, chunk = 0;
    if (tid == 0) {
        sh.b = n_batch;
        sh.base = 0;
    }
    for (int b0 = 0; b0 < n_batch; b0 += NT) {
        if (b0 > 0) __syncthreads();
        const uint32_t v = b0 == 0 ? v0 : (b0 + tid < n_batch ? (uint32_t)(tiles(request(b0 + tid)) * units_per_req) : 0u);
        const uint32_t incl = scan(v, chunk);
        if (b0 == 0) incl0 = incl;
        r.total += chunk;
    }
    r.ctas = (int)min(gridDim.x, r.total);
    r.lo = r.hi = r.total;
    if ((int)blockIdx.x < r.ctas) {
        r.lo = range_lo(r.total, blockIdx.x, r.ctas);
        r.hi = range_lo(r.total, blockIdx.x + 1, r.ctas);
    }
    uint32_t base = 0;
    for (int b0 = 0; b0 < n_batch; b0 += NT) {
        uint32_t v = v0, incl = incl0;
        if (n_batch > NT) {
            __syncthreads();
            if (b0 + tid < n_batch) mine = request(b0 + tid);
            v = b0 + tid < n_batch ? (uint32_t)(tiles(mine) * units_per_req) : 0u;
            incl = scan(v, chunk);
        }
        if (v > 0 && base + incl - v <= r.lo && r.lo < base + incl) {
            sh.b = b0 + tid;
            sh.base = base + incl - v;
            sh.req = mine;
        }
        base += chunk;
    }
    __syncthreads();
    r.b = sh.b;
    r.base = sh.base;
    r.req = sh.req;
    return r;
}

// ---- copy-engine feeder ----
// One lane's share of a 64-key tile of the paged prefix: lanes 0-15 copy K, 16-31 V, one run of rows inside one
// block each (blocks hold a multiple of 8 rows, so a tile spans at most 9 of them).
struct Piece {
    const uint8_t *src;  // first row of the run (bf16: its row group; Q8_0: its int8 row), or null
    int row, n;          // first row inside the tile, rows (multiple of 8)
    int rib;             // first row inside the block
};

// Block ids of a window of the request's table, in shared memory: read from global memory tile by tile, their
// latency bounded the feeder (one 16 KB tile per 0.9 us). Used by one warp.
constexpr int kTableWindow = 128;
struct TableWindow {
    int *blocks;  // [kTableWindow], -1 where the table's entry is no block
    int seq, lo, n;
    __device__ __forceinline__ void reset(int *mem) {
        blocks = mem;
        seq = -1;
        lo = n = 0;
    }
    // Entries [first, last] of the request, of which all up to `end` will be wanted in turn.
    __device__ __forceinline__ void want(const PoolView &p, int sq, int first, int last, int end, int lane) {
        if (sq == seq && first >= lo && last < lo + n) return;
        __syncwarp();
        seq = sq;
        lo = first;
        n = min(kTableWindow, end + 1 - first);
        for (int i = lane; i < n; i += 32) blocks[i] = lookup_block(p, sq, first + i);
        __syncwarp();
    }
};

template <int D, bool Q8>
__device__ __forceinline__ Piece find_piece(const TreeArgs &a, const Req &rq, int head, int key0, TableWindow &tw, int lane) {
    const PoolView &p = a.pool;
    const int valid = min(kTile, rq.n_prefix - key0), n8 = (valid + 7) & ~7;
    const int kv = lane >> 4, i = lane & 15;
    Piece pc;
    pc.src = nullptr;
    pc.row = pc.n = pc.rib = 0;
    if (valid <= 0) return pc;
    const int bt = p.block_tokens;
    auto block_of = [&](int pos) { return p.bt_shift >= 0 ? pos >> p.bt_shift : pos / bt; };
    const int blk0 = block_of(key0);
    tw.want(p, rq.seq, blk0, block_of(key0 + valid - 1), block_of(rq.n_prefix - 1), lane);
    const int e = blk0 + i;
    const int r0 = max(key0, e * bt), r1 = min(key0 + n8, (e + 1) * bt);
    if (r1 <= r0) return pc;
    const int blk = tw.blocks[e - tw.lo];
    if (blk < 0) return pc;
    pc.row = r0 - key0;
    pc.n = r1 - r0;
    pc.rib = r0 - e * bt;
    pc.src = p.prefix + prefix_tile_index(p, a.layer, blk, kv, head) * p.tile_bytes;
    return pc;
}

// Issue the lane's copies of a tile whose K lands at `dst_k` (completion on bar_k) and V at `dst_v`; lane 0 arrives on
// both. With WITH_V false only K is copied.
template <int D, bool Q8, bool WITH_V>
__device__ __forceinline__ void issue_piece(const TreeArgs &a, const Piece &pc, uint32_t dst_k, uint32_t dst_v,
                                            uint32_t bar_k, uint32_t bar_v, int lane) {
    using C = TileCfg<D, Q8>;
    using namespace sm100;
    constexpr int ROW = Q8 ? D : 2 * D, SROW = C::G32 * 2;  // bytes of a row, and of its scales
    const bool is_v = lane >= 16;
    const bool on = pc.src != nullptr && (WITH_V || !is_v);
    const uint32_t bytes = !on ? 0u : (uint32_t)(pc.n * (ROW + (Q8 ? SROW : 0)));
    const uint32_t kb = __reduce_add_sync(0xffffffffu, is_v ? 0u : bytes);
    const uint32_t vb = WITH_V ? __reduce_add_sync(0xffffffffu, is_v ? bytes : 0u) : 0u;
    if (lane == 0) {
        mbar_arrive_expect_tx(bar_k, kb);
        if (WITH_V) mbar_arrive_expect_tx(bar_v, vb);
    }
    __syncwarp();
    if (!on) return;
    const uint32_t dst = is_v ? dst_v : dst_k, bar = is_v ? bar_v : bar_k;
    bulk_g2s(dst + pc.row * ROW, pc.src + pc.rib * ROW, (uint32_t)(pc.n * ROW), bar);
    if (Q8)
        bulk_g2s(dst + C::SCALES + pc.row * SROW, pc.src + (int64_t)a.pool.block_tokens * D + pc.rib * SROW,
                 (uint32_t)(pc.n * SROW), bar);
}

// Bytes of a query row in shared memory, padded so that the operand loads below meet different banks: eight rows'
// 16-byte units (bf16), or two rows' 64 bytes (Q8_0).
template <int D, bool Q8>
__host__ __device__ constexpr int q_row_bytes() { return 2 * D + (Q8 ? 64 : 16); }

// Query operands of column steps 2 i and 2 i + 1 of the eight rows at `rows` (shared-memory address of the first).
template <int D, bool Q8>
__device__ __forceinline__ void load_q_steps(uint32_t rows, int i, int lane, uint32_t (&f)[4]) {
    if (Q8) {
        // in q_col's order a lane's columns of a 32-column group are 16 adjacent bytes
        const uint4 v = lds128(rows + (lane >> 2) * q_row_bytes<D, Q8>() + 64 * i + (lane & 3) * 16);
        f[0] = v.x;
        f[1] = v.y;
        f[2] = v.z;
        f[3] = v.w;
    } else {
        ldmatrix_x4(f, rows + (lane & 7) * q_row_bytes<D, Q8>() + 64 * i + (lane >> 3) * 16);
    }
}

// A warp's share (row `first`, first + step, ...) of n query rows to shared memory; `src(row)`: the row's elements,
// or null for a row of zeros. Wait with cp_async_wait_all().
template <int D, bool Q8, class Src>
__device__ __forceinline__ void stage_q_rows(uint32_t dst, int n, const uint16_t *any, int first, int step, int lane, Src src) {
    // 32 / U rows at a time, a lane one 16-byte unit (or two) of them
    constexpr int U = D / 8, UL = U < 32 ? U : 32, PER = 32 / UL;
    const int sub = lane / UL;
#pragma unroll 4
    for (int r = first * PER + sub; r < n; r += step * PER) {
        const uint16_t *row = src(r);
#pragma unroll
        for (int u = lane % UL; u < U; u += UL)
            if (sub < PER) cp_async_16_or_zero(dst + r * q_row_bytes<D, Q8>() + 16 * u, row ? row + 8 * u : any, row != nullptr);
    }
}

// ---- scores of one warp's 16 keys ----
// Column order of the matrix products. bf16 caches: natural. Q8_0 caches: step 2 g + i of group g (32
// columns) gives lane c of a quad the columns 32 g + 8 c + 4 i + {0, 1 | 2, 3}, so that a lane reads its
// 8 bytes of a group in one load; the query operands are taken in the same order, and a product does not depend
// on it.
template <bool Q8>
__device__ __forceinline__ int q_col(int step, int c, int half) {
    return Q8 ? 32 * (step >> 1) + 8 * c + 4 * (step & 1) + 2 * half : 16 * step + 2 * c + 8 * half;
}

// A operand of one 16-key x 16-column step of a bf16 tile: keys are its rows.
template <int D>
__device__ __forceinline__ void load_k_rows(uint32_t tile, int key0, int step, int lane, uint32_t (&a)[4]) {
    ldmatrix_x4(a, tile + bf16_off<D>(key0 + (lane & 15), 16 * step + (lane >> 4) * 8));
}

// A operand V^T: 16 columns of V (step `step`) are its rows, 16 keys its columns.
template <int D>
__device__ __forceinline__ void load_v_cols(uint32_t tile, int key0, int step, int lane, uint32_t (&a)[4]) {
    const int row = key0 + (lane & 7) + ((lane >> 4) << 3);
    ldmatrix_x4_trans(a, tile + bf16_off<D>(row, 16 * step + ((lane >> 3) & 1) * 8));
}

// An 8 x 8 matrix of 16-bit elements, transposed across the warp.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

}  // namespace decode
}  // namespace ekv
