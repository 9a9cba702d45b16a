// ekv_window.cuh -- what the kernels of windowed attention share: which slots a unit's rows see, and how tiles of them are fetched.
//
// Rows are (token, query head of the KV head's group), token-major. The row of the token at slot p sees the slots k <= p with
// k > p - window or k < sinks. A unit is a row tile of one request and KV head; what its rows see between them is the run
// [lo, hi) that ends with its last token, and the first tokens [0, front) before it where the window has left them behind.
// The two runs are taken as one sequence of keys (both start at a multiple of eight rows, as pages do), cut into tiles.
#pragma once

#include "ekv_decode.cuh"

namespace ekv {
namespace window {

// One request of the call: `n` rows' tokens from slot pos0 on; seq < 0: refused, its rows become 0.
struct WinReq {
    int seq, pos0, n, src;  // src: its first row in q and out
};

__device__ __forceinline__ WinReq load_win_req(const WindowArgs &a, int b, bool report) {
    WinReq r;
    r.seq = a.seq_ids[b];
    r.pos0 = a.dst_pos[b];
    r.n = min(max(a.n_rows[b], 0), a.max_rows);
    r.src = a.src_row[b];
    if (r.n == 0) return r;
    if (r.seq < 0 || r.seq >= a.pool.max_seqs) {
        if (report) report_error(a.pool.status, DEV_ERR_BAD_SEQ, b, r.seq, 14);
        r.seq = -1;
        return r;
    }
    const int len = a.pool.seq_lens[r.seq];
    if (r.pos0 < 0 || r.pos0 > len - r.n) {
        if (report) report_error(a.pool.status, DEV_ERR_BAD_POS, b, r.pos0, len);
        r.seq = -1;
    }
    return r;
}

// The keys of a unit whose tokens are at slots [first, last].
struct Span {
    int first, last;
    int front, lo, keys;  // keys in all: [0, front), then [lo, last]
    __device__ __forceinline__ Span(const WindowArgs &a, const WinReq &r, int token0, int token1) {
        first = r.pos0 + token0;
        last = r.pos0 + token1;
        lo = max(0, first - a.window + 1) & ~7;
        front = (int)(((uint32_t)min(a.sinks, lo) + 7u) & ~7u);
        if (front >= lo) front = lo = 0;
        keys = r.seq < 0 ? 0 : front + last + 1 - lo;
    }
    __device__ __forceinline__ int slot(int key) const { return key < front ? key : key - front + lo; }
    // Keys that no row sees, as runs begin and end at multiples of eight rows: n_hidden from `hidden` on, behind the first tokens and before
    // the first row's window.
    __device__ __forceinline__ int hidden(const WindowArgs &a) const { return min(a.sinks, max(0, first - a.window + 1) - lo + front); }
    __device__ __forceinline__ int n_hidden(const WindowArgs &a) const { return max(0, first - a.window + 1) - lo + front - hidden(a); }
    // Every row sees all of keys [key, key + n).
    __device__ __forceinline__ bool all_see(const WindowArgs &a, int key, int n) const {
        if (key < front) return key + n <= min(front, a.sinks);  // (lo > front: all before the first row)
        const int s = key - front + lo;
        return s + n - 1 <= first && (s > last - a.window || s + n <= a.sinks);
    }
};

__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// Which of keys [key, key + 32) the row at slot p sees, a bit each.
__device__ __forceinline__ uint32_t seen_bits(const WindowArgs &a, const Span &sp, int p, int key) {
    auto run = [&](int s) { return low_bits(p + 1 - s) & (low_bits(a.sinks - s) | ~low_bits(p - a.window + 1 - s)); };
    if (key >= sp.front) return run(key - sp.front + sp.lo);
    uint32_t bits = run(key);
    if (key + 32 > sp.front) {
        const uint32_t before = low_bits(sp.front - key);
        bits = (bits & before) | (run(key - sp.front + sp.lo) & ~before);
    }
    return bits;
}

// One lane's share of a tile of N keys: a run of rows inside one block (blocks hold a multiple of 8 rows, so there are at most
// N / 8 + 1 of them).
struct Run {
    const uint8_t *src;  // K of the block's head, or null
    int row, n, rib;     // first row inside the tile, rows (a multiple of 8), first row inside the block
};

// Lane `i` of a tile's runs, from key `key` on; block(e): the block of the request's table entry e, or -1; want(e0, e1): entries that
// will be asked for next, by the whole warp.
template <int N, class Want, class Block>
__device__ __forceinline__ Run find_run(const WindowArgs &a, const Span &sp, int head, int key, int i, Want want, Block block) {
    const PoolView &p = a.pool;
    Run r;
    r.src = nullptr;
    r.row = r.n = r.rib = 0;
    const int end = min(key + N, (sp.keys + 7) & ~7), bt = p.block_tokens;
    if (end <= key) return r;
    auto entry = [&](int slot) { return p.bt_shift >= 0 ? slot >> p.bt_shift : slot / bt; };
    int part_runs = 0;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const int k0 = part == 0 ? key : max(key, sp.front), k1 = part == 0 ? min(end, sp.front) : end;
        if (k1 <= k0) continue;
        const int s0 = sp.slot(k0), s1 = s0 + (k1 - k0), e0 = entry(s0), e1 = entry(s1 - 1);
        want(e0, e1);
        const int e = e0 + i - part_runs;
        if (i >= part_runs && e <= e1) {
            const int r0 = max(s0, e * bt), r1 = min(s1, (e + 1) * bt), blk = block(e);
            if (blk >= 0) {
                r.row = k0 - key + (r0 - s0);
                r.n = r1 - r0;
                r.rib = r0 - e * bt;
                r.src = p.prefix + prefix_tile_index(p, a.layer, blk, 0, head) * p.tile_bytes;
            }
        }
        part_runs += e1 - e0 + 1;
    }
    return r;
}

// floor(row / group) for the row of a unit (row * group < 2^32: checked at the call)
__device__ __forceinline__ int row_token(const WindowArgs &a, int row) { return a.group == 1 ? row : (int)__umulhi((uint32_t)row, a.group_mul); }

// Rows [row0, row0 + rows) of a request's KV head: their first and last tokens, among n.
__device__ __forceinline__ int last_token(const WindowArgs &a, int row0, int rows, int n) { return min(n - 1, row_token(a, row0 + rows - 1)); }

}  // namespace window
}  // namespace ekv
