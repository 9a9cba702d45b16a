// ekv_pages.cu -- copies of blocks for forked sequences, and rows that move together.
//
// Both only move bytes, so both are bound by DRAM, or by their few dependent reads where little moves.
//
// Copies: a block's rows in use are one run of bytes per tile (bf16), or two (8-bit rows, then their scales). A thread reads its
// 16-byte units once and writes them to every sibling's block. The children's table rows are written by the same launch: one
// upload per child and table took the host 5 us each.
//
// Compaction, slot i <- slot s_i with s_0 < s_1 < ...: as s_i >= i, a row that is overwritten by row i was wanted by rows up to
// i only. So a strip (layer, request, K|V, head) can be moved in place, chunk after chunk of rows: read the chunk into registers,
// meet, write it. A strip is one CTA's work, or a cluster's where the call has few strips.
#include <algorithm>

#include "ekv_decode.cuh"

namespace ekv {
namespace {

using namespace sm100;

constexpr int kThreads = 256;

// ---- copies and forks ----
template <int N>
struct PagesArgs {
    PoolView pool;
    int32_t n_copies, chunks;  // CTAs of a copy
    BlockCopy copy[N];
    int32_t dst[N];
    ForkedSeq child[N];
};

constexpr int kCopyLoads = 4;  // 16-byte units that a thread has on their way

// Grid: (chunk of the copy, copy), then one CTA per child.
template <int N, bool Q8>
__global__ void __launch_bounds__(kThreads) pages_kernel(const __grid_constant__ PagesArgs<N> a) {
    const PoolView &p = a.pool;
    decode::grid_wait();
    const int n_copy_ctas = a.n_copies * a.chunks;
    if ((int)blockIdx.x >= n_copy_ctas) {
        const ForkedSeq f = a.child[blockIdx.x - n_copy_ctas];
        const int w = p.max_blocks_per_seq;
        const int32_t *from = p.block_tables + (int64_t)f.parent * w;
        int32_t *to = p.block_tables + (int64_t)f.child * w;
        int32_t *to_write = p.write_tables + (int64_t)f.child * w, *from_write = p.write_tables + (int64_t)f.parent * w;
        for (int i = threadIdx.x; i < w; i += kThreads) {
            const bool shared = i < f.n_full;
            to[i] = shared ? from[i] : i == f.n_full ? f.tail : -1;
            to_write[i] = i == f.n_full ? f.tail : -1;
            if (shared) from_write[i] = -1;
        }
        if (threadIdx.x == 0) p.seq_lens[f.child] = f.n_tokens;
        return;
    }
    const int c = blockIdx.x / a.chunks, chunk = blockIdx.x - c * a.chunks;
    const BlockCopy job = a.copy[c];
    const int D = p.head_dim, heads = 2 * p.kv_heads;
    // units of a tile: rows, then (Q8) scales
    const int row_units = Q8 ? job.rows * D / 16 : job.rows * D / 8, units = row_units + (Q8 ? job.rows * (D / 32) / 8 : 0);
    const int scales = p.block_tokens * D, total = p.n_layers * heads * units;  // (below 2^30: checked at the call)
    auto offset = [&](int i) {  // in block 0
        const int tile = i / units, u = i - tile * units, layer = tile / heads, h = tile - layer * heads;
        return ((int64_t)layer * p.n_blocks * heads + h) * p.tile_bytes + (!Q8 || u < row_units ? 16 * u : scales + 16 * (u - row_units));
    };
    const int step = a.chunks * kThreads;  // (no more than what all units take)
    for (int i0 = chunk * kThreads + threadIdx.x; i0 < total; i0 += kCopyLoads * step) {
        uint4 v[kCopyLoads];
        int64_t at[kCopyLoads];
#pragma unroll
        for (int j = 0; j < kCopyLoads; ++j) {
            if (i0 + j * step >= total) continue;
            at[j] = offset(i0 + j * step);
            v[j] = *(const uint4 *)(p.prefix + at[j] + (int64_t)job.src * heads * p.tile_bytes);
        }
        for (int k = 0; k < job.n_dst; ++k) {
            uint8_t *to = p.prefix + (int64_t)a.dst[job.first + k] * heads * p.tile_bytes;
#pragma unroll
            for (int j = 0; j < kCopyLoads; ++j)
                if (i0 + j * step < total) *(uint4 *)(to + at[j]) = v[j];
        }
    }
}

template <int N>
int launch_pages_n(const PoolView &p, const BlockCopy *copies, int n_copies, const int32_t *dst, int n_dst, const ForkedSeq *children,
                   int n_children, int sms, cudaStream_t s) {
    static_assert(sizeof(PagesArgs<N>) <= 32000, "kernel parameters");
    PagesArgs<N> a;
    a.pool = p;
    a.n_copies = n_copies;
    int rows = 8;
    for (int i = 0; i < n_copies; ++i) {
        a.copy[i] = copies[i];
        rows = std::max(rows, copies[i].rows);
    }
    std::copy(dst, dst + n_dst, a.dst);
    std::copy(children, children + n_children, a.child);
    const int64_t units = (int64_t)p.n_layers * 2 * p.kv_heads * rows * p.head_dim / 8;
    const int64_t most = (units + kThreads * kCopyLoads - 1) / (kThreads * kCopyLoads);
    // a few units a thread, and no more CTAs than eight waves of them
    a.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(most, std::max<int64_t>(1, 64ll * sms / std::max(1, n_copies))));
    const int grid = n_copies * a.chunks + n_children;
    if (grid == 0) return EKV_OK;
    if (p.dtype == EKV_DTYPE_Q8_0) return decode::launch_after(pages_kernel<N, true>, grid, kThreads, 0, s, a);
    return decode::launch_after(pages_kernel<N, false>, grid, kThreads, 0, s, a);
}

// ---- compaction ----
constexpr int kRowLoads = 16;   // 16-byte units of a thread and chunk
constexpr int kListLoads = 8;   // entries of a thread and round, while rows stay
constexpr int kMaxCluster = 8;

// Where a row of the chunk comes from and goes to: tiles, and rows inside them. A row that stays has to < 0, and a source that
// may be read.
struct Move {
    const uint8_t *src;
    uint8_t *dst;
    int from, to;
};

// The scales of an 8-bit row (2 bytes for every 32 columns, adjacent), in one word of up to 16 bytes where their number allows.
__device__ __forceinline__ void load_row_scales(const uint8_t *src, int bytes, uint4 &v) {
    if (bytes == 16) {
        v = *(const uint4 *)src;
    } else if (bytes == 8) {
        *(uint2 *)&v = *(const uint2 *)src;
    } else {
        uint16_t h[8] = {};
#pragma unroll
        for (int g = 0; g < 7; ++g)
            if (2 * g < bytes) h[g] = ((const uint16_t *)src)[g];
        v = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6]);
    }
}
__device__ __forceinline__ void store_row_scales(uint8_t *dst, int bytes, const uint4 &v) {
    if (bytes == 16) {
        *(uint4 *)dst = v;
    } else if (bytes == 8) {
        *(uint2 *)dst = make_uint2(v.x, v.y);
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int g = 0; g < 7; ++g)
            if (2 * g < bytes) ((uint16_t *)dst)[g] = (uint16_t)(w[g >> 1] >> (16 * (g & 1)));
    }
}

// Grid: strips (layer, request, K|V, head) of `cluster` CTAs each. A thread resolves one row of the chunk after this one while
// its units are on their way, so that a chunk is one round trip to memory and not the four that slots, tables and rows are; its
// loads have no condition, and registers for all of them (two CTAs per SM): 8 requests of about 8 k slots, 4 layers, 8 heads of 128
// columns (1.36 GB read and written) take 225 us, 92% of the measured copy rate; with resolved slots in the same loop, conditions
// and four CTAs per SM 501; with 8 loads 250.
// EVEN: a row's units divide the threads, so that a thread keeps to one unit of its rows.
template <bool Q8, bool EVEN>
__global__ void __launch_bounds__(kThreads, 2) compact_kernel(const CompactArgs a, int cluster) {
    __shared__ int s_off[2];
    __shared__ Move s_moves[3][kThreads];  // (three: a thread may store a chunk while another resolves the one after the next)
    const PoolView &p = a.pool;
    if (threadIdx.x < 2) s_off[threadIdx.x] = INT32_MAX;
    __syncthreads();
    decode::grid_wait();
    const int strip = blockIdx.x / cluster, rank = blockIdx.x - strip * cluster, tid = threadIdx.x;
    const int heads = 2 * p.kv_heads, kvh = strip % heads, lb = strip / heads, b = lb % a.n_batch, layer = a.layer0 + lb / a.n_batch;
    const int seq = a.seq_ids[b], n = a.n_keep[b];
    // (every CTA of the cluster takes the same way)
    if (seq < 0 || seq >= p.max_seqs) {
        if (tid == 0) report_error(p.status, DEV_ERR_BAD_SEQ, b, seq, 12);
        return;
    }
    const int len = p.seq_lens[seq];
    if (n < 0 || n > a.slot_stride || n > len) {
        if (tid == 0) report_error(p.status, DEV_ERR_BAD_POS, b, n, len);
        return;
    }
    const int32_t *slots = a.slots + (int64_t)b * a.slot_stride;
    // Rows below `first` stay where they are. Every entry is looked at, up to the first that is not its own place: a list may be in order
    // again behind one that is not, and that one is to be reported. (60 000 rows of which 59 000 stay: 14 us; a search that trusted the
    // list took 5.)
    int first = 0;
    for (int round = 0; first < n; ++round) {
        int at[kListLoads], off = INT32_MAX;
#pragma unroll
        for (int j = 0; j < kListLoads; ++j) at[j] = tid + j * kThreads < n - first ? __ldg(slots + first + tid + j * kThreads) : -1;
#pragma unroll
        for (int j = kListLoads - 1; j >= 0; --j)
            if (tid + j * kThreads < n - first && at[j] != first + tid + j * kThreads) off = tid + j * kThreads;
        off = __reduce_min_sync(0xffffffffu, off);
        // (two, in turn: a thread may look at one round's while another is in the next)
        if (off != INT32_MAX && (tid & 31) == 0) atomicMin(&s_off[round & 1], off);
        __syncthreads();
        off = s_off[round & 1];
        if (off != INT32_MAX) {
            first += off;
            break;
        }
        first += min(n - first, kThreads * kListLoads);
    }
    const int D = p.head_dim, wlog = decode::log2_of(p.swz_bytes), bt = p.block_tokens;
    const int per = Q8 ? D / 16 : D / 8;  // units of a row
    // rows of a CTA and chunk: what its loads hold, or an even share of few rows
    const int rows = min(min(kThreads, kThreads * kRowLoads / per), (n - first + cluster - 1) / cluster), per_chunk = cluster * rows;
    uint8_t *const base = p.prefix + ((int64_t)layer * p.n_blocks * heads + kvh) * p.tile_bytes;
    const int64_t block_bytes = (int64_t)heads * p.tile_bytes;
    auto resolve = [&](int64_t row0) {
        Move m{base, nullptr, 0, -1};
        const int64_t i = row0 + (int64_t)rank * rows + tid;
        if (tid >= rows || i >= n) return m;
        const int from = __ldg(slots + i), before = i > 0 ? __ldg(slots + i - 1) : -1;
        if (from < i || from >= len || from <= before) {
            report_error(p.status, DEV_ERR_BAD_POS, seq, from, len);
            return m;
        }
        if (from == i) return m;
        const int fb = from / bt, tb = (int)i / bt;
        const int bs = lookup_block(p, seq, fb), bd = lookup_block_to_write(p, seq, tb);
        if (bs < 0 || bd < 0) return m;
        m.src = base + bs * block_bytes;
        m.dst = base + bd * block_bytes;
        m.from = from - fb * bt;
        m.to = (int)i - tb * bt;
        return m;
    };
    auto offset = [&](int rib, int u) { return Q8 ? q8_qs_off(rib, 16 * u, D) : decode::bf16_off_any(rib, 8 * u, D, wlog); };
    const uint32_t per_mul = (uint32_t)(((1ull << 32) + per - 1) / per);  // (items are below 2^12: exact; not for per == 1)
    auto row_of = [&](int item) { return per == 1 ? item : (int)__umulhi((uint32_t)item, per_mul); };
    const int r_even = row_of(tid), u_even = tid - r_even * per, r_step = kThreads / per;
    auto place = [&](int j, int &r, int &u) {
        if (EVEN) {
            r = r_even + j * r_step;
            u = u_even;
        } else {
            r = row_of(tid + j * kThreads);
            u = tid + j * kThreads - r * per;
        }
    };
    s_moves[0][tid] = resolve(first);
    __syncthreads();
    int buf = 0;
    for (int64_t row0 = first; row0 < n; row0 += per_chunk) {
        const Move *moves = s_moves[buf];
        uint4 v[kRowLoads], sc;
#pragma unroll
        for (int j = 0; j < kRowLoads; ++j) {
            int r, u;
            place(j, r, u);
            const Move &m = moves[r & (kThreads - 1)];  // (past the last row: any, its source may be read)
            v[j] = *(const uint4 *)(m.src + offset(m.from, u));
        }
        if (Q8) load_row_scales(moves[tid].src + bt * D + moves[tid].from * (D / 16), D / 16, sc);
        const int next = buf == 2 ? 0 : buf + 1;
        if (row0 + per_chunk < n) s_moves[next][tid] = resolve(row0 + per_chunk);
        // everything of the chunk has been read
        if (cluster > 1) cluster_sync();
        else __syncthreads();
#pragma unroll
        for (int j = 0; j < kRowLoads; ++j) {
            if (j * kThreads >= rows * per) break;
            int r, u;
            place(j, r, u);
            if (r < rows && moves[r].to >= 0) *(uint4 *)(moves[r].dst + offset(moves[r].to, u)) = v[j];
        }
        if (Q8 && tid < rows && moves[tid].to >= 0) store_row_scales(moves[tid].dst + bt * D + moves[tid].to * (D / 16), D / 16, sc);
        buf = next;
    }
}

}  // namespace

int launch_pages(const PoolView &p, const BlockCopy *copies, int n_copies, const int32_t *dst, int n_dst, const ForkedSeq *children,
                 int n_children, int sms, cudaStream_t s) {
    if (std::max({n_copies, n_dst, n_children}) <= 16) return launch_pages_n<16>(p, copies, n_copies, dst, n_dst, children, n_children, sms, s);
    return launch_pages_n<kMaxForks>(p, copies, n_copies, dst, n_dst, children, n_children, sms, s);
}

int launch_compact(const CompactArgs &a, int sms, cudaStream_t s) {
    const int64_t strips = (int64_t)a.n_layers * a.n_batch * 2 * a.pool.kv_heads;
    int c = 1;
    while (c < kMaxCluster && strips * 8 * c <= 5 * sms) c *= 2;
    if (strips * c > INT32_MAX) return EKV_ERR_INVALID_ARG;
    const bool q8 = a.pool.dtype == EKV_DTYPE_Q8_0, even = kThreads % (a.pool.head_dim / (q8 ? 16 : 8)) == 0;
    const auto kernel = q8 ? (even ? compact_kernel<true, true> : compact_kernel<true, false>)
                           : (even ? compact_kernel<false, true> : compact_kernel<false, false>);
    return decode::launch_clusters_after(c, kernel, (unsigned)(strips * c), kThreads, 0, s, a, c);
}

}  // namespace ekv
