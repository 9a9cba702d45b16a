// ekv_capi.cpp -- C-ABI entry points and the host-side pool manager (block allocator, block
// tables, sequence slots). Every entry point validates its arguments before enqueuing work.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <new>
#include <set>

#include "ekv_internal.h"

using ekv::PoolView;

namespace {

constexpr size_t kAlign = 1024;

size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

bool valid_seq(const ekv_pool *p, int32_t id) {
    return p && id >= 0 && id < p->cfg.max_seqs && p->seqs[(size_t)id].live;
}

int32_t blocks_for(const ekv_pool *p, int32_t n_tokens) {
    return (n_tokens + p->cfg.block_tokens - 1) / p->cfg.block_tokens;
}

// The predicted range within the sequence's length (empty ranges normalised to [0, 0)).
void clamp_pred(ekv_pool::Seq &q) {
    q.pred_hi = std::min(q.pred_hi, q.n_tokens);
    q.pred_lo = std::min(q.pred_lo, q.pred_hi);
    if (q.pred_hi <= q.pred_lo) q.pred_lo = q.pred_hi = 0;
}

void mark_dirty(ekv_pool *p, int32_t id) {
    p->dirty[(size_t)id] = 1;
    p->any_dirty = true;
}

// Blocks in and out of sequences: a block is free again when its last holder lets it go.
int32_t take_lowest_block(ekv_pool *p) {
    const int32_t b = p->free_blocks.take();
    p->holders[(size_t)b] = 1;
    return b;
}
void release_block(ekv_pool *p, int32_t b) {
    const int32_t left = --p->holders[(size_t)b];
    if (left == 0) p->free_blocks.insert(b);
    if (left == 1) p->unshared = p->any_dirty = true;  // its last holder may write it again: known at the next sync
}

// Makes the pool's device current for one entry point and restores the caller's current device when
// the entry point returns (a library inside a host such as a ggml backend must not move its device).
class DeviceScope {
  public:
    explicit DeviceScope(const ekv_pool *p) {
        if (p->cfg.device < 0) {
            rc_ = EKV_ERR_UNSUPPORTED;  // host-only pool
            return;
        }
        if (cudaGetDevice(&prev_) != cudaSuccess) {
            cudaGetLastError();
            rc_ = EKV_ERR_CUDA;
            return;
        }
        if (prev_ != p->cfg.device && cudaSetDevice(p->cfg.device) != cudaSuccess) {
            rc_ = EKV_ERR_CUDA;
            return;
        }
        switched_ = prev_ != p->cfg.device;
    }
    ~DeviceScope() {
        if (switched_) cudaSetDevice(prev_);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
    int rc() const { return rc_; }

  private:
    int prev_ = 0;
    int rc_ = EKV_OK;
    bool switched_ = false;
};

}  // namespace

namespace ekv {
static std::atomic<unsigned long long> g_launches{0};
void note_launches(int n) { g_launches.fetch_add((unsigned long long)n, std::memory_order_relaxed); }
static std::atomic<int> g_debug_stall{0};
bool take_debug_stall() { return g_debug_stall.exchange(0, std::memory_order_relaxed) != 0; }
}  // namespace ekv

extern "C" {

const char *ekv_version(void) { return "ekv 0.1 (sm_100a)"; }

uint64_t ekv_launch_count(void) { return ekv::g_launches.load(std::memory_order_relaxed); }

int ekv_debug_expire_wait(int32_t enable) {
    ekv::g_debug_stall.store(enable ? 1 : 0, std::memory_order_relaxed);
    return EKV_OK;
}

const char *ekv_strerror(int code) {
    switch (code) {
        case EKV_OK: return "ok";
        case EKV_ERR_INVALID_ARG: return "invalid argument";
        case EKV_ERR_CUDA: return "CUDA runtime error";
        case EKV_ERR_POOL_EXHAUSTED: return "pool exhausted";
        case EKV_ERR_NO_SEQ: return "unknown sequence";
        case EKV_ERR_RANGE: return "position or length out of range";
        case EKV_ERR_UNSUPPORTED: return "unsupported shape or dtype";
        case EKV_ERR_DEVICE: return "kernel reported a bad index";
        case EKV_ERR_TIMEOUT: return "kernel wait budget ran out";
        case EKV_ERR_ALLOC: return "allocation failed";
        default: return "unknown error";
    }
}

int ekv_pool_create(const ekv_pool_config *cfg, ekv_pool **out) {
    if (!cfg || !out) return EKV_ERR_INVALID_ARG;
    *out = nullptr;
    const ekv_pool_config c = *cfg;
    if (c.dtype != EKV_DTYPE_BF16 && c.dtype != EKV_DTYPE_Q8_0) return EKV_ERR_UNSUPPORTED;
    if (c.block_tokens <= 0 || c.block_tokens % 8 || c.block_tokens > 256) return EKV_ERR_INVALID_ARG;
    if (c.head_dim <= 0 || c.head_dim > 256 || c.head_dim % 16) return EKV_ERR_UNSUPPORTED;
    if (c.dtype == EKV_DTYPE_Q8_0 && c.head_dim % 32) return EKV_ERR_UNSUPPORTED;
    if (c.n_blocks <= 0 || c.kv_heads <= 0 || c.n_layers <= 0 || c.max_seqs <= 0 ||
        c.max_blocks_per_seq <= 0 || c.suffix_tokens < 0 || c.suffix_tokens > 4096)
        return EKV_ERR_INVALID_ARG;

    ekv_pool *p = new (std::nothrow) ekv_pool();
    if (!p) return EKV_ERR_ALLOC;
    p->cfg = c;
    const DeviceScope dev_scope(p);
    if (c.device >= 0 && dev_scope.rc()) {
        delete p;
        return dev_scope.rc();
    }
    p->sms = 148;
    if (c.device >= 0 && cudaDeviceGetAttribute(&p->sms, cudaDevAttrMultiProcessorCount, c.device) != cudaSuccess) {
        delete p;
        return EKV_ERR_CUDA;
    }
    PoolView &v = p->view;
    v.dtype = c.dtype;
    v.block_tokens = c.block_tokens;
    v.n_blocks = c.n_blocks;
    v.kv_heads = c.kv_heads;
    v.head_dim = c.head_dim;
    v.n_layers = c.n_layers;
    v.max_seqs = c.max_seqs;
    v.max_blocks_per_seq = c.max_blocks_per_seq;
    v.suffix_rows = (c.suffix_tokens + 15) / 16 * 16;
    v.swz_bytes = ekv::swizzle_bytes_for(c.head_dim);
    try {
        p->holders.assign((size_t)c.n_blocks, 0);
    } catch (const std::bad_alloc &) {
        delete p;
        return EKV_ERR_ALLOC;
    }
    v.bt_shift = -1;
    for (int sh = 0; sh < 16; ++sh)
        if ((1 << sh) == c.block_tokens) v.bt_shift = sh;
    v.tile_bytes = c.dtype == EKV_DTYPE_BF16
                       ? (int64_t)c.block_tokens * c.head_dim * 2
                       : (int64_t)c.block_tokens * c.head_dim + (int64_t)c.block_tokens * (c.head_dim / 32) * 2;
    v.suffix_tile_bytes = (int64_t)v.suffix_rows * c.head_dim * 2;

    p->bytes_prefix = align_up((size_t)c.n_layers * c.n_blocks * 2 * c.kv_heads * (size_t)v.tile_bytes, kAlign);
    p->bytes_suffix = align_up((size_t)c.n_layers * c.max_seqs * 2 * c.kv_heads * (size_t)v.suffix_tile_bytes, kAlign);
    const size_t bytes_tables = align_up((size_t)c.max_seqs * c.max_blocks_per_seq * 4, kAlign);
    const size_t bytes_lens = align_up((size_t)c.max_seqs * 4, kAlign);
    const size_t bytes_status = kAlign;
    p->bytes_total = p->bytes_prefix + p->bytes_suffix + bytes_tables + bytes_lens + bytes_status;

    if (c.device < 0) {
        // Host-only pool: block tables and sequences without device memory (for testing the
        // allocator where no GPU is present). Data operations on it fail with EKV_ERR_UNSUPPORTED.
        p->free_blocks.fill(c.n_blocks);
        p->seqs.resize((size_t)c.max_seqs);
        p->dirty.assign((size_t)c.max_seqs, 0);
        p->free_seq_ids.fill(c.max_seqs);
        *out = p;
        return EKV_OK;
    }
    if (cudaMalloc(&p->dev_base, p->bytes_total) != cudaSuccess) {
        cudaGetLastError();
        delete p;
        return EKV_ERR_ALLOC;
    }
    if (cudaMallocHost((void **)&p->h_status, 4 * sizeof(int32_t)) != cudaSuccess) {
        cudaGetLastError();
        cudaFree(p->dev_base);
        delete p;
        return EKV_ERR_ALLOC;
    }
    if (cudaMemset(p->dev_base, 0, p->bytes_total) != cudaSuccess) {
        cudaFreeHost(p->h_status);
        cudaFree(p->dev_base);
        delete p;
        return EKV_ERR_CUDA;
    }
    uint8_t *base = (uint8_t *)p->dev_base;
    v.prefix = base;
    v.suffix = base + p->bytes_prefix;
    v.block_tables = (int32_t *)(base + p->bytes_prefix + p->bytes_suffix);
    v.write_tables = v.block_tables;
    v.seq_lens = (int32_t *)(base + p->bytes_prefix + p->bytes_suffix + bytes_tables);
    v.status = (int32_t *)(base + p->bytes_prefix + p->bytes_suffix + bytes_tables + bytes_lens);

    p->free_blocks.fill(c.n_blocks);
    p->seqs.resize((size_t)c.max_seqs);
    p->dirty.assign((size_t)c.max_seqs, 0);
    p->free_seq_ids.fill(c.max_seqs);
    if (cudaDeviceSynchronize() != cudaSuccess) {
        cudaFreeHost(p->h_status);
        cudaFree(p->dev_base);
        delete p;
        return EKV_ERR_CUDA;
    }
    *out = p;
    return EKV_OK;
}

int ekv_pool_destroy(ekv_pool *p) {
    if (!p) return EKV_ERR_INVALID_ARG;
    if (p->cfg.device < 0) {
        delete p;
        return EKV_OK;
    }
    const DeviceScope dev_scope(p);
    cudaDeviceSynchronize();
    if (p->h_status) cudaFreeHost(p->h_status);
    if (p->dev_base) cudaFree(p->dev_base);
    if (p->dev_write_tables) cudaFree(p->dev_write_tables);
    delete p;
    return EKV_OK;
}

int ekv_pool_get_info(const ekv_pool *p, ekv_pool_info *info) {
    if (!p || !info) return EKV_ERR_INVALID_ARG;
    info->bytes_total = p->bytes_total;
    info->bytes_prefix = p->bytes_prefix;
    info->bytes_suffix = p->bytes_suffix;
    info->block_bytes = (size_t)p->view.tile_bytes * 2 * p->cfg.kv_heads;
    info->free_blocks = (int32_t)p->free_blocks.size();
    info->live_seqs = p->cfg.max_seqs - (int32_t)p->free_seq_ids.size();
    info->prefix_base = p->view.prefix;
    info->suffix_base = p->view.suffix;
    info->block_tables = p->view.block_tables;
    info->seq_lens = p->view.seq_lens;
    return EKV_OK;
}

int ekv_pool_status(ekv_pool *p, int32_t *code, ekv_stream_t stream) {
    if (!p || !code) return EKV_ERR_INVALID_ARG;
    if (p->cfg.device < 0) {
        *code = EKV_OK;
        return EKV_OK;
    }
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    cudaStream_t s = (cudaStream_t)stream;
    if (cudaMemcpyAsync(p->h_status, p->view.status, 4 * sizeof(int32_t), cudaMemcpyDeviceToHost, s) != cudaSuccess ||
        cudaMemsetAsync(p->view.status, 0, 4 * sizeof(int32_t), s) != cudaSuccess ||
        cudaStreamSynchronize(s) != cudaSuccess)
        return EKV_ERR_CUDA;
    *code = p->h_status[0];
    return EKV_OK;
}

// Upload the rows of changed sequences, adjacent ones together.
static int upload_dirty(ekv_pool *p, cudaStream_t s) {
    const int32_t W = p->cfg.max_blocks_per_seq;
    // Pageable sources: cudaMemcpyAsync stages them before returning, so the host vectors may
    // change right after this call.
    std::vector<int32_t> rows, lens;
    for (int32_t id = 0; id < p->cfg.max_seqs;) {
        if (!p->dirty[(size_t)id]) {
            ++id;
            continue;
        }
        int32_t end = id;
        rows.clear();
        lens.clear();
        for (; end < p->cfg.max_seqs && p->dirty[(size_t)end]; ++end) {
            const ekv_pool::Seq &q = p->seqs[(size_t)end];
            rows.insert(rows.end(), q.blocks.begin(), q.blocks.end());
            rows.resize((size_t)(end - id + 1) * W, -1);
            lens.push_back(q.live ? q.n_tokens : 0);
        }
        const size_t n = (size_t)(end - id), at = (size_t)id * W;
        if (cudaMemcpyAsync(p->view.block_tables + at, rows.data(), n * W * 4, cudaMemcpyHostToDevice, s) != cudaSuccess ||
            cudaMemcpyAsync(p->view.seq_lens + id, lens.data(), n * 4, cudaMemcpyHostToDevice, s) != cudaSuccess)
            return EKV_ERR_CUDA;
        if (p->dev_write_tables) {
            for (int32_t &b : rows)
                if (b >= 0 && p->holders[(size_t)b] > 1) b = -1;
            if (cudaMemcpyAsync(p->dev_write_tables + at, rows.data(), n * W * 4, cudaMemcpyHostToDevice, s) != cudaSuccess)
                return EKV_ERR_CUDA;
        }
        std::fill(p->dirty.begin() + id, p->dirty.begin() + end, (uint8_t)0);
        id = end;
    }
    return EKV_OK;
}

int ekv_pool_sync(ekv_pool *p, ekv_stream_t stream) {
    if (!p) return EKV_ERR_INVALID_ARG;
    if (!p->any_dirty || p->cfg.device < 0) return EKV_OK;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    if (p->unshared && p->dev_write_tables) {
        for (int32_t id = 0; id < p->cfg.max_seqs; ++id)
            if (p->seqs[(size_t)id].live && p->seqs[(size_t)id].forked) p->dirty[(size_t)id] = 1;
    }
    try {
        if (const int rc = upload_dirty(p, (cudaStream_t)stream)) return rc;
    } catch (const std::bad_alloc &) {
        return EKV_ERR_ALLOC;
    }
    p->any_dirty = p->unshared = false;
    return EKV_OK;
}

int ekv_seq_create(ekv_pool *p, int32_t *seq_id) {
    if (!p || !seq_id) return EKV_ERR_INVALID_ARG;
    if (p->free_seq_ids.empty()) return EKV_ERR_POOL_EXHAUSTED;
    const int32_t id = p->free_seq_ids.take();
    ekv_pool::Seq &q = p->seqs[(size_t)id];
    q.live = true;
    q.forked = false;
    q.n_tokens = 0;
    q.blocks.clear();
    q.pred_lo = q.pred_hi = 0;
    mark_dirty(p, id);
    *seq_id = id;
    return EKV_OK;
}

int ekv_seq_free(ekv_pool *p, int32_t id) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    ekv_pool::Seq &q = p->seqs[(size_t)id];
    for (int32_t b : q.blocks) release_block(p, b);
    q.blocks.clear();
    q.n_tokens = 0;
    q.pred_lo = q.pred_hi = 0;
    q.live = false;
    p->free_seq_ids.insert(id);
    mark_dirty(p, id);
    return EKV_OK;
}

int ekv_seq_resize(ekv_pool *p, int32_t id, int32_t n_tokens) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    if (n_tokens < 0) return EKV_ERR_INVALID_ARG;
    ekv_pool::Seq &q = p->seqs[(size_t)id];
    const int32_t need = blocks_for(p, n_tokens);
    if (need > p->cfg.max_blocks_per_seq) return EKV_ERR_RANGE;
    const int32_t have = (int32_t)q.blocks.size();
    if (need > have) {
        if ((int32_t)p->free_blocks.size() < need - have) return EKV_ERR_POOL_EXHAUSTED;
        for (int32_t i = have; i < need; ++i) q.blocks.push_back(take_lowest_block(p));
    } else {
        for (int32_t i = need; i < have; ++i) release_block(p, q.blocks[(size_t)i]);
        q.blocks.resize((size_t)need);
    }
    q.n_tokens = n_tokens;
    clamp_pred(q);
    mark_dirty(p, id);
    return EKV_OK;
}

int ekv_seq_set_blocks(ekv_pool *p, int32_t id, const int32_t *blocks, int32_t n_blocks,
                       int32_t n_tokens) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    if ((!blocks && n_blocks) || n_blocks < 0 || n_tokens < 0) return EKV_ERR_INVALID_ARG;
    if (n_blocks > p->cfg.max_blocks_per_seq || blocks_for(p, n_tokens) > n_blocks) return EKV_ERR_RANGE;
    ekv_pool::Seq &q = p->seqs[(size_t)id];
    // Every requested block must be free or already owned by this sequence, and distinct.
    std::set<int32_t> own(q.blocks.begin(), q.blocks.end()), seen;
    for (int32_t i = 0; i < n_blocks; ++i) {
        const int32_t b = blocks[i];
        if (b < 0 || b >= p->cfg.n_blocks) return EKV_ERR_INVALID_ARG;
        if (!seen.insert(b).second) return EKV_ERR_INVALID_ARG;
        if (!own.count(b) && !p->free_blocks.has(b)) return EKV_ERR_POOL_EXHAUSTED;
    }
    for (int32_t b : q.blocks) release_block(p, b);
    q.blocks.assign(blocks, blocks + n_blocks);
    for (int32_t b : q.blocks) {
        p->free_blocks.erase(b);
        ++p->holders[(size_t)b];
    }
    q.n_tokens = n_tokens;
    q.pred_lo = q.pred_hi = 0;
    mark_dirty(p, id);
    return EKV_OK;
}

int ekv_seq_evict_front(ekv_pool *p, int32_t id, int32_t n_blocks) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    ekv_pool::Seq &q = p->seqs[(size_t)id];
    if (n_blocks < 0 || n_blocks > (int32_t)q.blocks.size()) return EKV_ERR_RANGE;
    for (int32_t i = 0; i < n_blocks; ++i) release_block(p, q.blocks[(size_t)i]);
    q.blocks.erase(q.blocks.begin(), q.blocks.begin() + n_blocks);
    const int32_t shift = n_blocks * p->cfg.block_tokens;
    q.n_tokens = std::max(0, q.n_tokens - shift);
    q.pred_lo = std::max(0, q.pred_lo - shift);
    q.pred_hi = std::max(0, q.pred_hi - shift);
    clamp_pred(q);
    mark_dirty(p, id);
    return EKV_OK;
}

int ekv_seq_drop_blocks(ekv_pool *p, int32_t id, int32_t first, int32_t n_blocks) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    ekv_pool::Seq &q = p->seqs[(size_t)id];
    const int32_t have = (int32_t)q.blocks.size();
    if (first < 0 || n_blocks < 0 || first > have || n_blocks > have - first) return EKV_ERR_RANGE;
    // (a table reaches no further than 2^31 tokens: ekv_seq_resize and ekv_seq_set_blocks count them in 32 bits)
    const int64_t bt = p->cfg.block_tokens;
    const int32_t lo = (int32_t)std::min<int64_t>(q.n_tokens, first * bt), hi = (int32_t)std::min<int64_t>(q.n_tokens, (first + n_blocks) * bt);
    if (q.pred_hi > q.pred_lo && q.pred_lo < hi && q.pred_hi > lo) return EKV_ERR_UNSUPPORTED;  // predicted tokens: ekv_seq_clear_pred
    for (int32_t i = first; i < first + n_blocks; ++i) release_block(p, q.blocks[(size_t)i]);
    q.blocks.erase(q.blocks.begin() + first, q.blocks.begin() + first + n_blocks);
    q.n_tokens -= hi - lo;
    if (q.pred_lo >= hi) {
        q.pred_lo -= hi - lo;
        q.pred_hi -= hi - lo;
    }
    clamp_pred(q);
    mark_dirty(p, id);
    return EKV_OK;
}

// The writers' own tables, from the first fork on: which blocks a sequence alone holds.
static int make_write_tables(ekv_pool *p) {
    if (p->cfg.device < 0 || p->dev_write_tables) return EKV_OK;
    const size_t bytes = (size_t)p->cfg.max_seqs * p->cfg.max_blocks_per_seq * 4;
    if (cudaMalloc((void **)&p->dev_write_tables, bytes) != cudaSuccess) {
        cudaGetLastError();
        p->dev_write_tables = nullptr;
        return EKV_ERR_ALLOC;
    }
    p->bytes_total += bytes;
    p->view.write_tables = p->dev_write_tables;
    for (int32_t id = 0; id < p->cfg.max_seqs; ++id) p->dirty[(size_t)id] = 1;
    p->any_dirty = true;
    return EKV_OK;
}

// The copies count the 16-byte units of a block, all layers, in 32 bits.
static bool copies_too_large(const ekv_pool *p) {
    return (int64_t)p->cfg.n_layers * 2 * p->cfg.kv_heads > (1ll << 34) / p->view.tile_bytes;
}

static int fork_sequences(ekv_pool *p, int32_t n, const int32_t *parents, const int32_t *n_tokens, int32_t *children, cudaStream_t s) {
    const int32_t bt = p->cfg.block_tokens;
    const bool device = p->cfg.device >= 0;
    std::vector<ekv::BlockCopy> copies;
    std::vector<ekv::ForkedSeq> forks;
    std::vector<int32_t> dst;
    copies.reserve(ekv::kMaxForks);
    forks.reserve(ekv::kMaxForks);
    dst.reserve(ekv::kMaxForks);
    for (int32_t i = 0, id = 0; i < n; ++i, ++id) {
        id = p->free_seq_ids.next(id);
        p->seqs[(size_t)id].blocks.reserve((size_t)blocks_for(p, n_tokens[i]));
    }
    if (device) {
        if (const int rc = make_write_tables(p)) return rc;
        // The kernel reads the parents' tables and writes the children's. (Blocks that are no longer shared may wait: so marked,
        // they are refused to writers, no more.)
        auto mark = [&](uint8_t to) {
            for (int32_t i = 0, id = 0; i < n; ++i, ++id) p->dirty[(size_t)(id = p->free_seq_ids.next(id))] = to;
        };
        mark(0);
        if (const int rc = upload_dirty(p, s)) {
            p->any_dirty = true;
            mark(1);
            return rc;
        }
        p->any_dirty = p->unshared;
    }
    for (int32_t i = 0; i < n; ++i) {
        ekv_pool::Seq &from = p->seqs[(size_t)parents[i]];
        const int32_t full = n_tokens[i] / bt, rest = n_tokens[i] % bt;
        int32_t tail = -1;
        const int32_t id = p->free_seq_ids.take();
        ekv_pool::Seq &q = p->seqs[(size_t)id];
        std::vector<int32_t> &blocks = q.blocks;
        blocks.assign(from.blocks.begin(), from.blocks.begin() + full);
        for (int32_t b : blocks) ++p->holders[(size_t)b];
        if (rest) {
            tail = take_lowest_block(p);
            blocks.push_back(tail);
            const int32_t src = from.blocks[(size_t)full], rows = (rest + 7) / 8 * 8;
            if (!copies.empty() && copies.back().src == src && copies.back().rows == rows) ++copies.back().n_dst;  // a sibling
            else copies.push_back({src, rows, (int32_t)dst.size(), 1});
            dst.push_back(tail);
        }
        q.live = q.forked = from.forked = true;
        q.n_tokens = n_tokens[i];
        q.pred_lo = q.pred_hi = 0;
        children[i] = id;
        if (!device) {
            mark_dirty(p, id);
            continue;
        }
        forks.push_back({parents[i], id, full, tail, n_tokens[i]});
        if ((int32_t)forks.size() < ekv::kMaxForks && i + 1 < n) continue;
        const int rc = ekv::launch_pages(p->view, copies.data(), (int)copies.size(), dst.data(), (int)dst.size(), forks.data(),
                                         (int)forks.size(), p->sms, s);
        if (rc) {  // back to the parents alone; the next sync writes their tables again
            for (int32_t k = 0; k <= i; ++k) {
                ekv_seq_free(p, children[k]);
                mark_dirty(p, parents[k]);
                children[k] = -1;
            }
            return rc;
        }
        copies.clear();
        forks.clear();
        dst.clear();
    }
    return EKV_OK;
}

int ekv_seq_fork(ekv_pool *p, int32_t n, const int32_t *parents, const int32_t *n_tokens, int32_t *children, ekv_stream_t stream) {
    if (!p || n < 0 || (n > 0 && (!parents || !n_tokens || !children))) return EKV_ERR_INVALID_ARG;
    if (copies_too_large(p)) return EKV_ERR_UNSUPPORTED;
    int64_t tails = 0;
    for (int32_t i = 0; i < n; ++i) {
        if (!valid_seq(p, parents[i])) return EKV_ERR_NO_SEQ;
        if (n_tokens[i] < 0 || n_tokens[i] > p->seqs[(size_t)parents[i]].n_tokens) return EKV_ERR_RANGE;
        tails += n_tokens[i] % p->cfg.block_tokens != 0;
    }
    if ((int64_t)p->free_seq_ids.size() < n || (int64_t)p->free_blocks.size() < tails) return EKV_ERR_POOL_EXHAUSTED;
    if (n == 0) return EKV_OK;
    const DeviceScope dev_scope(p);
    if (p->cfg.device >= 0 && dev_scope.rc()) return dev_scope.rc();
    try {
        return fork_sequences(p, n, parents, n_tokens, children, (cudaStream_t)stream);
    } catch (const std::bad_alloc &) {  // (every allocation comes before the first change, but for the freed sequences' marks)
        for (int32_t i = 0, id = 0; i < n; ++i, ++id) mark_dirty(p, id = p->free_seq_ids.next(id));
        return EKV_ERR_ALLOC;
    }
}

int ekv_seq_own(ekv_pool *p, int32_t id, int32_t pos0, int32_t n_tokens, ekv_stream_t stream) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    if (copies_too_large(p)) return EKV_ERR_UNSUPPORTED;
    ekv_pool::Seq &q = p->seqs[(size_t)id];
    const int32_t bt = p->cfg.block_tokens, have = (int32_t)q.blocks.size();
    if (pos0 < 0 || n_tokens < 0 || (int64_t)pos0 + n_tokens > (int64_t)have * bt) return EKV_ERR_RANGE;
    if (n_tokens == 0) return ekv_pool_sync(p, stream);
    const int32_t first = pos0 / bt, last = (int32_t)(((int64_t)pos0 + n_tokens - 1) / bt);
    int32_t shared = 0;
    for (int32_t i = first; i <= last; ++i) shared += p->holders[(size_t)q.blocks[(size_t)i]] > 1;
    // (what was shared once may still be marked so on the device, and the sequence may have grown)
    if (shared == 0) return ekv_pool_sync(p, stream);
    if ((int32_t)p->free_blocks.size() < shared) return EKV_ERR_POOL_EXHAUSTED;
    const DeviceScope dev_scope(p);
    if (p->cfg.device >= 0 && dev_scope.rc()) return dev_scope.rc();
    int rc = EKV_OK;
    int32_t at = first;
    while (at <= last && !rc) {
        // some copies at a time: their launch comes first, so that a failure leaves the sequence as it was
        ekv::BlockCopy copies[ekv::kMaxForks];
        int32_t dst[ekv::kMaxForks], entry[ekv::kMaxForks];
        int n = 0;
        int32_t next = -1;
        for (; at <= last && n < ekv::kMaxForks; ++at) {
            if (p->holders[(size_t)q.blocks[(size_t)at]] <= 1) continue;
            copies[n] = {q.blocks[(size_t)at], bt, n, 1};
            entry[n] = at;
            dst[n++] = next = p->free_blocks.next(next + 1);
        }
        if (p->cfg.device >= 0 && n > 0)
            rc = ekv::launch_pages(p->view, copies, n, dst, n, nullptr, 0, p->sms, (cudaStream_t)stream);
        for (int i = 0; i < n && !rc; ++i) {
            q.blocks[(size_t)entry[i]] = take_lowest_block(p);  // (dst[i])
            release_block(p, copies[i].src);
        }
        mark_dirty(p, id);
    }
    if (p->cfg.device >= 0 && !rc) rc = ekv_pool_sync(p, stream);
    return rc;
}

int ekv_seq_append_tokens(ekv_pool *p, int32_t id, int32_t n_tokens, int32_t pred) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    if (n_tokens < 0) return EKV_ERR_INVALID_ARG;
    ekv_pool::Seq &q = p->seqs[(size_t)id];
    const int32_t old = q.n_tokens;
    const bool has_pred = q.pred_hi > q.pred_lo;
    if (pred && has_pred && q.pred_hi != old) return EKV_ERR_UNSUPPORTED;  // a second predicted range
    if ((int64_t)old + n_tokens > INT32_MAX) return EKV_ERR_RANGE;
    if (const int rc = ekv_seq_resize(p, id, old + n_tokens)) return rc;
    if (pred && n_tokens > 0) {
        if (!has_pred) q.pred_lo = old;
        q.pred_hi = old + n_tokens;
    }
    return EKV_OK;
}

int ekv_seq_clear_pred(ekv_pool *p, int32_t id) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    ekv_pool::Seq &q = p->seqs[(size_t)id];
    if (q.pred_hi <= q.pred_lo) return EKV_OK;
    const int32_t bt = p->cfg.block_tokens, lo = q.pred_lo, hi = q.pred_hi;
    if (hi == q.n_tokens) {
        q.pred_lo = q.pred_hi = 0;
        return ekv_seq_resize(p, id, lo);  // truncation cannot fail
    }
    if (lo % bt || hi % bt) return EKV_ERR_UNSUPPORTED;
    for (int32_t i = lo / bt; i < hi / bt; ++i) release_block(p, q.blocks[(size_t)i]);
    q.blocks.erase(q.blocks.begin() + lo / bt, q.blocks.begin() + hi / bt);
    q.n_tokens -= hi - lo;
    q.pred_lo = q.pred_hi = 0;
    mark_dirty(p, id);
    return EKV_OK;
}

int ekv_seq_restore(ekv_pool *p, int32_t id, int32_t n_tokens) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    ekv_pool::Seq &q = p->seqs[(size_t)id];
    if (n_tokens < 0 || n_tokens > q.n_tokens) return EKV_ERR_RANGE;
    return ekv_seq_resize(p, id, q.n_tokens - n_tokens);
}

int ekv_seq_get_pred(const ekv_pool *p, int32_t id, int32_t *lo, int32_t *hi) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    const ekv_pool::Seq &q = p->seqs[(size_t)id];
    if (lo) *lo = q.pred_lo;
    if (hi) *hi = q.pred_hi;
    return EKV_OK;
}

int ekv_seq_get(const ekv_pool *p, int32_t id, int32_t *n_tokens, int32_t *n_blocks,
                int32_t *blocks, int32_t cap) {
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    const ekv_pool::Seq &q = p->seqs[(size_t)id];
    if (n_tokens) *n_tokens = q.n_tokens;
    if (n_blocks) *n_blocks = (int32_t)q.blocks.size();
    if (blocks) {
        const int32_t n = std::min(cap, (int32_t)q.blocks.size());
        for (int32_t i = 0; i < n; ++i) blocks[i] = q.blocks[(size_t)i];
    }
    return EKV_OK;
}

int ekv_append(ekv_pool *p, int32_t layer, int32_t n_batch, const int32_t *seq_ids,
               const int32_t *dst_pos, const int32_t *n_rows, const int32_t *src_row,
               int32_t max_rows, const void *k, const void *v, ekv_stream_t stream) {
    if (!p || !seq_ids || !dst_pos || !n_rows || !src_row || !k || !v) return EKV_ERR_INVALID_ARG;
    if (layer < 0 || layer >= p->cfg.n_layers || n_batch < 0 || max_rows < 0) return EKV_ERR_INVALID_ARG;
    if (n_batch == 0 || max_rows == 0) return EKV_OK;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    return ekv::launch_append(p->view, layer, n_batch, seq_ids, dst_pos, n_rows, src_row, max_rows,
                              k, v, (cudaStream_t)stream);
}

int ekv_append_suffix(ekv_pool *p, int32_t layer, int32_t n_batch, const int32_t *seq_ids,
                      int32_t n_rows, const void *k, const void *v, ekv_stream_t stream) {
    if (!p || !seq_ids || !k || !v) return EKV_ERR_INVALID_ARG;
    if (layer < 0 || layer >= p->cfg.n_layers || n_batch < 0 || n_rows < 0) return EKV_ERR_INVALID_ARG;
    if (n_rows > p->cfg.suffix_tokens) return EKV_ERR_RANGE;
    if (n_batch == 0 || n_rows == 0) return EKV_OK;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    return ekv::launch_append_suffix(p->view, layer, n_batch, seq_ids, n_rows, k, v, (cudaStream_t)stream);
}

int ekv_gather(ekv_pool *p, int32_t layer, int32_t id, int32_t pos0, int32_t n_rows, int32_t format,
               void *k_out, void *v_out, ekv_stream_t stream) {
    if (!p || !k_out || !v_out) return EKV_ERR_INVALID_ARG;
    if (format != EKV_GATHER_NATIVE && format != EKV_GATHER_F32) return EKV_ERR_INVALID_ARG;
    if (layer < 0 || layer >= p->cfg.n_layers) return EKV_ERR_INVALID_ARG;
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    if (pos0 < 0 || n_rows < 0 || pos0 + n_rows > p->seqs[(size_t)id].n_tokens) return EKV_ERR_RANGE;
    if (n_rows == 0) return EKV_OK;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    return ekv::launch_gather(p->view, layer, id, pos0, n_rows, format, k_out, v_out, (cudaStream_t)stream);
}

int ekv_gather_suffix(ekv_pool *p, int32_t layer, int32_t id, int32_t n_rows, int32_t format,
                      void *k_out, void *v_out, ekv_stream_t stream) {
    if (!p || !k_out || !v_out) return EKV_ERR_INVALID_ARG;
    if (format != EKV_GATHER_NATIVE && format != EKV_GATHER_F32) return EKV_ERR_INVALID_ARG;
    if (layer < 0 || layer >= p->cfg.n_layers) return EKV_ERR_INVALID_ARG;
    if (!valid_seq(p, id)) return EKV_ERR_NO_SEQ;
    if (n_rows < 0 || n_rows > p->cfg.suffix_tokens) return EKV_ERR_RANGE;
    if (n_rows == 0) return EKV_OK;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    return ekv::launch_gather_suffix(p->view, layer, id, n_rows, format, k_out, v_out, (cudaStream_t)stream);
}

static int fill_attn_args(ekv_pool *p, const ekv_attn_params *prm, const void *q, void *out,
                          ekv::AttnArgs &a) {
    if (!p || !prm || !q || !out || !prm->seq_ids) return EKV_ERR_INVALID_ARG;
    if (((uintptr_t)q | (uintptr_t)out) & 15) return EKV_ERR_INVALID_ARG;  // 16-byte vector loads/stores
    const ekv_pool_config &c = p->cfg;
    if (prm->layer < 0 || prm->layer >= c.n_layers) return EKV_ERR_INVALID_ARG;
    if (prm->n_batch <= 0 || prm->q_tokens <= 0 || prm->q_heads <= 0) return EKV_ERR_INVALID_ARG;
    if (prm->q_heads % c.kv_heads) return EKV_ERR_INVALID_ARG;
    if (prm->suffix_len < 0 || prm->suffix_len > c.suffix_tokens) return EKV_ERR_RANGE;
    if (prm->out_dtype != EKV_DTYPE_BF16 && prm->out_dtype != EKV_DTYPE_F32) return EKV_ERR_UNSUPPORTED;
    if (!(prm->scale > 0.0f) || !std::isfinite(prm->scale)) return EKV_ERR_INVALID_ARG;
    if ((prm->mask_flags & EKV_MASK_BLOCK_CAUSAL) &&
        (prm->chunk_tokens <= 0 || prm->chunk_stride < prm->chunk_tokens || prm->window_chunks <= 0))
        return EKV_ERR_INVALID_ARG;
    if ((prm->mask_flags & (EKV_MASK_SPAN_ONLY | EKV_MASK_SPAN_EXCLUDE)) && (!prm->span_begin || !prm->span_end))
        return EKV_ERR_INVALID_ARG;
    if ((prm->mask_flags & (EKV_MASK_FLEX_SELF | EKV_MASK_FLEX_CROSS)) &&
        (!prm->flex_meta || prm->flex_stride < 0 || (prm->n_batch > 1 && prm->flex_stride == 0) || prm->flex_q0 < 0 ||
         prm->flex_k0 < 0 || prm->flex_window < 0))
        return EKV_ERR_INVALID_ARG;
    if (prm->mask_flags & ~(EKV_MASK_SUFFIX_CAUSAL | EKV_MASK_SUFFIX_PREFIX_LM | EKV_MASK_SPAN_ONLY | EKV_MASK_SPAN_EXCLUDE |
                            EKV_MASK_BLOCK_CAUSAL | EKV_MASK_FLEX_SELF | EKV_MASK_FLEX_CROSS))
        return EKV_ERR_INVALID_ARG;
    a = ekv::AttnArgs{};
    a.pool = p->view;
    a.layer = prm->layer;
    a.n_batch = prm->n_batch;
    a.q_tokens = prm->q_tokens;
    a.q_heads = prm->q_heads;
    a.group = prm->q_heads / c.kv_heads;
    a.scale_log2 = prm->scale * 1.4426950408889634f;
    a.mask_flags = prm->mask_flags;
    a.chunk_tokens = prm->chunk_tokens;
    a.chunk_stride = prm->chunk_stride;
    a.window_chunks = prm->window_chunks;
    a.q_chunk0 = prm->q_chunk0;
    a.suffix_len = prm->suffix_len;
    a.out_dtype = prm->out_dtype;
    a.use_prefix = prm->use_prefix;
    a.seq_ids = prm->seq_ids;
    a.prefix_len = prm->prefix_len;
    a.prefix_valid = prm->prefix_valid;
    a.span_begin = prm->span_begin;
    a.span_end = prm->span_end;
    a.flex_meta = prm->flex_meta;
    a.flex_stride = prm->flex_stride;
    a.flex_q0 = prm->flex_q0;
    a.flex_k0 = prm->flex_k0;
    a.flex_window = prm->flex_window;
    a.q = (const uint16_t *)q;
    a.out = out;
    a.n_splits = 1;
    a.wait_budget = ekv::kDefaultWaitBudget;
    a.debug_stall = 0;
    return EKV_OK;
}

size_t ekv_attention_workspace_size(const ekv_pool *p, const ekv_attn_params *prm) {
    if (!p || !prm) return 0;
    return ekv::attention_tc_workspace(p->view, *prm, p->cfg.max_blocks_per_seq * p->cfg.block_tokens, p->sms);
}

int ekv_attention_algo(ekv_pool *p, const ekv_attn_params *prm, const void *q, void *out,
                       void *workspace, size_t workspace_bytes, int32_t algo, ekv_stream_t stream) {
    ekv::AttnArgs a;
    const int rc = fill_attn_args(p, prm, q, out, a);
    if (rc) return rc;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    if (algo == EKV_ALGO_SIMT) return ekv::launch_attention_simt(a, (cudaStream_t)stream);
    if (algo != EKV_ALGO_TC && algo != EKV_ALGO_TC_PAIR && algo != EKV_ALGO_TC_CTA && algo != EKV_ALGO_TC_PAIR64 &&
        algo != EKV_ALGO_TC_HEADS)
        return EKV_ERR_INVALID_ARG;
    const size_t need = ekv::attention_tc_workspace(p->view, *prm, p->cfg.max_blocks_per_seq * p->cfg.block_tokens, p->sms);
    if (workspace && ((uintptr_t)workspace & 15)) return EKV_ERR_INVALID_ARG;
    if (workspace && need && workspace_bytes >= need) {
        // The split count and the workspace carve-up are recomputed by the launcher.
        a.ws_o = (float *)workspace;
        a.n_splits = 0;  // 0 = let the launcher choose from the workspace it was given
    }
    const ekv::TcKernel k = algo == EKV_ALGO_TC_PAIR     ? ekv::TcKernel::Pair
                            : algo == EKV_ALGO_TC_CTA    ? ekv::TcKernel::OneCta
                            : algo == EKV_ALGO_TC_PAIR64 ? ekv::TcKernel::Pair64
                            : algo == EKV_ALGO_TC_HEADS  ? ekv::TcKernel::Heads
                                                         : ekv::TcKernel::Auto;
    return ekv::launch_attention_tc(a, (cudaStream_t)stream, k);
}

int ekv_attention(ekv_pool *p, const ekv_attn_params *prm, const void *q, void *out, void *workspace,
                  size_t workspace_bytes, ekv_stream_t stream) {
    return ekv_attention_algo(p, prm, q, out, workspace, workspace_bytes, EKV_ALGO_TC, stream);
}

int ekv_project_qkv_rope(ekv_pool *p, int32_t layer, int32_t n_batch, const int32_t *seq_ids, int32_t tokens,
                         int32_t q_heads, int32_t hidden, const void *x, const void *wq, const void *wk, const void *wv,
                         const int32_t *positions, float rope_base, void *q_out, void *k_out, void *v_out,
                         ekv_stream_t stream) {
    if (!p || !x || !wq || !wk || !wv || !positions || !q_out) return EKV_ERR_INVALID_ARG;
    if ((k_out == nullptr) != (v_out == nullptr)) return EKV_ERR_INVALID_ARG;
    const ekv_pool_config &c = p->cfg;
    if (layer < 0 || layer >= c.n_layers || n_batch <= 0 || tokens <= 0 || q_heads <= 0 || q_heads % c.kv_heads)
        return EKV_ERR_INVALID_ARG;
    if (hidden <= 0 || hidden % 64 || !(rope_base > 0.0f) || !std::isfinite(rope_base)) return EKV_ERR_INVALID_ARG;
    if ((int64_t)n_batch * tokens > INT_MAX / 2) return EKV_ERR_INVALID_ARG;
    if (((uintptr_t)x | (uintptr_t)wq | (uintptr_t)wk | (uintptr_t)wv | (uintptr_t)q_out | (uintptr_t)k_out |
         (uintptr_t)v_out) & 15)
        return EKV_ERR_INVALID_ARG;
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return EKV_ERR_UNSUPPORTED;
    if (!k_out) {  // into the suffix slots
        if (!seq_ids || c.suffix_tokens == 0) return EKV_ERR_INVALID_ARG;
        if (tokens > c.suffix_tokens) return EKV_ERR_RANGE;
    }
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    return ekv::launch_project_qkv(p->view, layer, n_batch, seq_ids, tokens, q_heads, hidden, x, wq, wk, wv, positions,
                                   rope_base, q_out, k_out, v_out, (cudaStream_t)stream);
}

int ekv_append_suffix_attention(ekv_pool *p, const ekv_attn_params *prm, const void *k_suffix,
                                const void *v_suffix, const void *q, void *out, void *workspace,
                                size_t workspace_bytes, ekv_stream_t stream) {
    if (!p || !prm || !k_suffix || !v_suffix) return EKV_ERR_INVALID_ARG;
    if (prm->layer < 0 || prm->layer >= p->cfg.n_layers || prm->n_batch < 0 || prm->suffix_len < 0)
        return EKV_ERR_INVALID_ARG;
    if (prm->suffix_len > p->cfg.suffix_tokens) return EKV_ERR_RANGE;
    if (((uintptr_t)k_suffix | (uintptr_t)v_suffix) & 15) return EKV_ERR_INVALID_ARG;
    if (p->cfg.suffix_tokens == 0) return EKV_ERR_INVALID_ARG;
    ekv::AttnArgs a;
    if (const int rc = fill_attn_args(p, prm, q, out, a)) return rc;
    if (workspace && ((uintptr_t)workspace & 15)) return EKV_ERR_INVALID_ARG;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    const cudaStream_t s = (cudaStream_t)stream;
    if (p->cfg.head_dim == 256) {
        // the CTA-pair kernel reads the suffix from the caller's buffers; the slot is not written
        a.k_sfx = (const uint16_t *)k_suffix;
        a.v_sfx = (const uint16_t *)v_suffix;
    } else if (prm->suffix_len > 0) {
        const int rc = ekv::launch_append_suffix(p->view, prm->layer, prm->n_batch, prm->seq_ids, prm->suffix_len,
                                                 k_suffix, v_suffix, s);
        if (rc) return rc;
    }
    const size_t need = ekv::attention_tc_workspace(p->view, *prm, p->cfg.max_blocks_per_seq * p->cfg.block_tokens, p->sms);
    if (workspace && need && workspace_bytes >= need) {
        a.ws_o = (float *)workspace;
        a.n_splits = 0;
    }
    return ekv::launch_attention_tc(a, s, ekv::TcKernel::Auto);
}

// Checks of a rotary append, which also fills in the strides of adjacent rows.
static int check_rope_append(const ekv_pool *p, const ekv_rope *rope, int32_t layer, int32_t n_batch, const int32_t *seq_ids,
                             const int32_t *dst_pos, const int32_t *n_rows, const int32_t *src_row, int32_t max_rows,
                             const int32_t *positions, int32_t q_heads, const void *q, int64_t &q_stride, const void *q_out,
                             const void *k, const void *v, int64_t &kv_stride) {
    if (!p || !rope || !n_rows || !src_row || !positions) return EKV_ERR_INVALID_ARG;
    if ((q == nullptr) != (q_out == nullptr) || (k == nullptr) != (v == nullptr) || (!q && !k)) return EKV_ERR_INVALID_ARG;
    if (k && (!seq_ids || !dst_pos)) return EKV_ERR_INVALID_ARG;
    const ekv_pool_config &c = p->cfg;
    if (layer < 0 || layer >= c.n_layers || n_batch < 0 || n_batch > 65535 || max_rows < 0) return EKV_ERR_INVALID_ARG;
    if (q && q_heads <= 0) return EKV_ERR_INVALID_ARG;
    if (ekv::rope_dims(rope) > c.head_dim) return EKV_ERR_INVALID_ARG;
    const int64_t q_row = q ? (int64_t)q_heads * c.head_dim : 0, kv_row = (int64_t)c.kv_heads * c.head_dim;
    if (q_stride == 0) q_stride = q_row;
    if (kv_stride == 0) kv_stride = kv_row;
    if ((q && (q_stride < q_row || q_stride % 8)) || (k && (kv_stride < kv_row || kv_stride % 8))) return EKV_ERR_INVALID_ARG;
    if (q && q == q_out && q_stride != q_row) return EKV_ERR_INVALID_ARG;
    if (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v) & 15) return EKV_ERR_INVALID_ARG;
    return EKV_OK;
}

int ekv_rope_append(ekv_pool *p, const ekv_rope *rope, int32_t layer, int32_t n_batch, const int32_t *seq_ids,
                    const int32_t *dst_pos, const int32_t *n_rows, const int32_t *src_row, int32_t max_rows,
                    const int32_t *positions, int32_t q_heads, const void *q, int64_t q_stride, void *q_out,
                    const void *k, const void *v, int64_t kv_stride, ekv_stream_t stream) {
    if (const int rc = check_rope_append(p, rope, layer, n_batch, seq_ids, dst_pos, n_rows, src_row, max_rows, positions, q_heads, q,
                                         q_stride, q_out, k, v, kv_stride))
        return rc;
    if (n_batch == 0 || max_rows == 0) return EKV_OK;
    if (ekv::rope_device(rope) != p->cfg.device) return EKV_ERR_INVALID_ARG;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    return ekv::launch_rope_append(p->view, rope, layer, n_batch, seq_ids, dst_pos, n_rows, src_row, max_rows, positions,
                                   q_heads, q, q_stride, q_out, k, v, kv_stride, p->sms, (cudaStream_t)stream);
}

int ekv_norm_rope_append(ekv_pool *p, const ekv_rope *rope, const ekv_head_norm *norm, int32_t layer, int32_t n_batch,
                         const int32_t *seq_ids, const int32_t *dst_pos, const int32_t *n_rows, const int32_t *src_row,
                         int32_t max_rows, const int32_t *positions, int32_t q_heads, const void *q, int64_t q_stride, void *q_out,
                         const void *k, const void *v, int64_t kv_stride, ekv_stream_t stream) {
    if (!norm || !(norm->eps >= 0.0f) || !std::isfinite(norm->eps) || !std::isfinite(norm->weight_offset)) return EKV_ERR_INVALID_ARG;
    if (((uintptr_t)norm->q_weight | (uintptr_t)norm->k_weight) & 15) return EKV_ERR_INVALID_ARG;
    if (const int rc = check_rope_append(p, rope, layer, n_batch, seq_ids, dst_pos, n_rows, src_row, max_rows, positions, q_heads, q,
                                         q_stride, q_out, k, v, kv_stride))
        return rc;
    if (norm->weight_dtype != EKV_DTYPE_F32 && norm->weight_dtype != EKV_DTYPE_BF16) return EKV_ERR_UNSUPPORTED;
    if (n_batch == 0 || max_rows == 0) return EKV_OK;
    if (ekv::rope_device(rope) != p->cfg.device) return EKV_ERR_INVALID_ARG;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    return ekv::launch_norm_rope_append(p->view, rope, norm, layer, n_batch, seq_ids, dst_pos, n_rows, src_row, max_rows, positions,
                                   q_heads, q, q_stride, q_out, k, v, kv_stride, p->sms, (cudaStream_t)stream);
}

// Rows of a KV head times its query heads, EKV_MAX_DRAFT * group^2, are 32-bit in the kernels.
static bool group_too_large(int group) { return group >= 8192; }
static_assert(EKV_MAX_DRAFT * 8191ll * 8191 < 1ll << 32, "rows times query heads");

// Checks what attention and key weights share, and the longest prefix to expect (which only sizes grids).
static int fill_tree_args(const ekv_pool *p, const ekv_tree_params *prm, const void *q, ekv::TreeArgs &a, int &max_len) {
    if (!p || !prm || !q || !prm->seq_ids) return EKV_ERR_INVALID_ARG;
    const ekv_pool_config &c = p->cfg;
    if (prm->layer < 0 || prm->layer >= c.n_layers || prm->n_batch <= 0 || prm->n_draft <= 0 || prm->q_heads <= 0 ||
        prm->q_heads % c.kv_heads)
        return EKV_ERR_INVALID_ARG;
    if (prm->n_draft > EKV_MAX_DRAFT) return EKV_ERR_RANGE;
    if (prm->max_prefix < 0) return EKV_ERR_INVALID_ARG;
    const float log2e = 1.4426950408889634f;
    if (!(prm->scale > 0.0f) || !std::isfinite(prm->scale * log2e) || !(prm->softcap >= 0.0f) || !std::isfinite(prm->softcap * log2e))
        return EKV_ERR_INVALID_ARG;
    const float cap_in = prm->softcap > 0.0f ? prm->scale / prm->softcap : 0.0f;
    if (!std::isfinite(cap_in)) return EKV_ERR_INVALID_ARG;  // (0 * inf for a score of 0)
    if (((uintptr_t)q | ((uintptr_t)prm->ancestors << 1)) & 15) return EKV_ERR_INVALID_ARG;
    if (c.head_dim != 48 && c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return EKV_ERR_UNSUPPORTED;
    a = ekv::TreeArgs{};
    a.pool = p->view;
    a.layer = prm->layer;
    a.n_batch = prm->n_batch;
    a.n_draft = prm->n_draft;
    a.q_heads = prm->q_heads;
    a.group = prm->q_heads / c.kv_heads;
    a.group_mul = (uint32_t)(((1ull << 32) + a.group - 1) / a.group);  // (not used at 1, where it is 2^32)
    if (group_too_large(a.group)) return EKV_ERR_UNSUPPORTED;
    a.scale_log2 = prm->scale * log2e;
    a.cap_log2 = prm->softcap * log2e;
    a.cap_in = cap_in;
    a.seq_ids = prm->seq_ids;
    a.prefix_len = prm->prefix_len;
    a.n_nodes = prm->n_nodes;
    a.ancestors = prm->ancestors;
    a.q = (const uint16_t *)q;
    max_len = 0;
    for (const ekv_pool::Seq &s : p->seqs)
        if (s.live) max_len = std::max(max_len, s.n_tokens);
    if (prm->max_prefix > 0) max_len = std::min(max_len, prm->max_prefix);
    return EKV_OK;
}

size_t ekv_tree_attention_workspace_size(const ekv_pool *p, const ekv_tree_params *prm) {
    if (!p || !prm || prm->n_batch <= 0 || prm->n_draft <= 0 || prm->n_draft > EKV_MAX_DRAFT || prm->q_heads <= 0 ||
        prm->q_heads % p->cfg.kv_heads || group_too_large(prm->q_heads / p->cfg.kv_heads))
        return 0;
    return ekv::tree_workspace(p->view, prm->n_batch, prm->n_draft, prm->q_heads, prm->softcap > 0.0f, p->sms);
}

int ekv_tree_attention(ekv_pool *p, const ekv_tree_params *prm, const void *q, const void *k_draft, const void *v_draft,
                       void *out, float *lse, void *workspace, size_t workspace_bytes, ekv_stream_t stream) {
    ekv::TreeArgs a;
    int max_len = 0;
    if (const int rc = fill_tree_args(p, prm, q, a, max_len)) return rc;
    if (!k_draft || !v_draft || !out) return EKV_ERR_INVALID_ARG;
    if (((uintptr_t)k_draft | (uintptr_t)v_draft | (uintptr_t)out | (uintptr_t)workspace) & 15) return EKV_ERR_INVALID_ARG;
    if ((uintptr_t)lse & 3) return EKV_ERR_INVALID_ARG;
    if (prm->out_dtype != EKV_DTYPE_BF16 && prm->out_dtype != EKV_DTYPE_F32) return EKV_ERR_UNSUPPORTED;
    a.k_draft = (const uint16_t *)k_draft;
    a.v_draft = (const uint16_t *)v_draft;
    a.out = out;
    a.lse = lse;
    a.out_dtype = prm->out_dtype;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    return ekv::launch_tree_attention(a, max_len, workspace, workspace_bytes, p->sms, (cudaStream_t)stream);
}

int ekv_key_weights(ekv_pool *p, const ekv_tree_params *prm, const void *q, const float *lse, float *weights,
                    int64_t weight_stride, float decay, ekv_stream_t stream) {
    ekv::TreeArgs a;
    int max_len = 0;
    if (const int rc = fill_tree_args(p, prm, q, a, max_len)) return rc;
    if (!lse || !weights || weight_stride < 0 || !std::isfinite(decay)) return EKV_ERR_INVALID_ARG;
    if (((uintptr_t)lse | (uintptr_t)weights) & 3) return EKV_ERR_INVALID_ARG;
    a.lse = const_cast<float *>(lse);
    a.weights = weights;
    a.weight_stride = weight_stride;
    a.decay = decay;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    return ekv::launch_key_weights(a, max_len, p->sms, (cudaStream_t)stream);
}

// Rows of a KV head times its query heads are 32-bit in the kernels, and so are a KV head's rows.
static bool window_rows_fit(const ekv_window_params *prm, const ekv_pool *p) {
    const int64_t group = prm->q_heads / p->cfg.kv_heads;
    return group < 8192 && (prm->max_rows + 256ll) * group < (1ll << 32) / group && prm->max_rows * group < INT32_MAX - 512;
}

size_t ekv_window_attention_workspace_size(const ekv_pool *p, const ekv_window_params *prm) {
    if (!p || !prm || prm->n_batch <= 0 || prm->max_rows <= 0 || prm->q_heads <= 0 || prm->q_heads % p->cfg.kv_heads ||
        !window_rows_fit(prm, p))
        return 0;
    return ekv::window_workspace(p->view, prm->n_batch, prm->max_rows, prm->q_heads, p->sms);
}

int ekv_window_attention(ekv_pool *p, const ekv_window_params *prm, const void *q, int64_t q_stride, void *out, void *workspace,
                         size_t workspace_bytes, ekv_stream_t stream) {
    if (!p || !prm || !q || !out || q == out || !prm->seq_ids || !prm->dst_pos || !prm->n_rows || !prm->src_row) return EKV_ERR_INVALID_ARG;
    const ekv_pool_config &c = p->cfg;
    if (prm->layer < 0 || prm->layer >= c.n_layers || prm->n_batch < 0 || prm->max_rows < 0 || prm->q_heads <= 0 || prm->q_heads % c.kv_heads)
        return EKV_ERR_INVALID_ARG;
    if (prm->window < 0 || prm->sinks < 0 || prm->max_len < 0) return EKV_ERR_INVALID_ARG;
    const float log2e = 1.4426950408889634f;
    if (!(prm->scale > 0.0f) || !std::isfinite(prm->scale * log2e)) return EKV_ERR_INVALID_ARG;
    const int64_t row = (int64_t)prm->q_heads * c.head_dim;
    if (q_stride == 0) q_stride = row;
    if (q_stride < row || q_stride % 8) return EKV_ERR_INVALID_ARG;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15) return EKV_ERR_INVALID_ARG;
    if (((uintptr_t)prm->seq_ids | (uintptr_t)prm->dst_pos | (uintptr_t)prm->n_rows | (uintptr_t)prm->src_row) & 3) return EKV_ERR_INVALID_ARG;
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return EKV_ERR_UNSUPPORTED;
    if (!window_rows_fit(prm, p)) return EKV_ERR_UNSUPPORTED;
    if (prm->n_batch == 0 || prm->max_rows == 0) return EKV_OK;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    ekv::WindowArgs a{};
    a.pool = p->view;
    a.layer = prm->layer;
    a.n_batch = prm->n_batch;
    a.q_heads = prm->q_heads;
    a.group = prm->q_heads / c.kv_heads;
    a.group_mul = (uint32_t)(((1ull << 32) + a.group - 1) / a.group);  // (not used at 1, where it is 2^32)
    a.max_rows = prm->max_rows;
    // (no sequence is that long, and slots less the window stay inside 32 bits for every key of a row's tiles)
    constexpr int32_t all = INT32_MAX - 1024;
    a.window = prm->window > 0 ? std::min(prm->window, all) : all;
    a.sinks = prm->sinks;
    a.scale_log2 = prm->scale * log2e;
    a.seq_ids = prm->seq_ids;
    a.dst_pos = prm->dst_pos;
    a.n_rows = prm->n_rows;
    a.src_row = prm->src_row;
    a.q = (const uint16_t *)q;
    a.q_stride = q_stride;
    a.out = (uint16_t *)out;
    int max_len = 0;
    for (const ekv_pool::Seq &s : p->seqs)
        if (s.live) max_len = std::max(max_len, s.n_tokens);
    if (prm->max_len > 0) max_len = std::min(max_len, prm->max_len);
    return ekv::launch_window_attention(a, max_len, workspace, workspace_bytes, p->sms, (cudaStream_t)stream);
}

int ekv_evict_by_weight(ekv_pool *p, const ekv_evict_params *prm, ekv_stream_t stream) {
    if (!p || !prm || !prm->seq_ids || !prm->weights || !prm->kept) return EKV_ERR_INVALID_ARG;
    const ekv_pool_config &c = p->cfg;
    if (prm->layer0 < 0 || prm->n_layers <= 0 || prm->n_layers > c.n_layers - prm->layer0 || prm->n_batch <= 0)
        return EKV_ERR_INVALID_ARG;
    if (prm->keep <= 0 || prm->first < 0 || prm->recent < 0 || (int64_t)prm->first + prm->recent > prm->keep)
        return EKV_ERR_INVALID_ARG;
    if (prm->keep > INT32_MAX - 4096) return EKV_ERR_RANGE;  // the kernels count slots past it in 32 bits
    if (prm->weight_stride < 0 || ((prm->weights_out || prm->positions_out) && prm->out_stride < prm->keep))
        return EKV_ERR_INVALID_ARG;
    // in place only where slot i is the same entry on both sides
    if (((const float *)prm->weights_out == prm->weights || (prm->positions && prm->positions_out == prm->positions)) &&
        prm->out_stride != prm->weight_stride)
        return EKV_ERR_INVALID_ARG;
    if (((uintptr_t)prm->weights | (uintptr_t)prm->kept | (uintptr_t)prm->positions | (uintptr_t)prm->weights_out |
         (uintptr_t)prm->positions_out) & 3)
        return EKV_ERR_INVALID_ARG;
    // Which sequences the call means is known on the device, where one that is too long is reported. Here the call is
    // refused when its distinct sequences cannot all be short enough.
    int max_len = 0, fit = 0, too_long = 0;
    for (const ekv_pool::Seq &s : p->seqs) {
        if (!s.live) continue;
        max_len = std::max(max_len, s.n_tokens);
        (s.n_tokens > EKV_MAX_EVICT_TOKENS ? too_long : fit)++;
    }
    if (too_long > 0 && prm->n_batch > fit) return EKV_ERR_RANGE;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    ekv::EvictArgs a{};
    a.pool = p->view;
    a.layer0 = prm->layer0;
    a.n_layers = prm->n_layers;
    a.n_batch = prm->n_batch;
    a.keep = prm->keep;
    a.first = prm->first;
    a.recent = prm->recent;
    a.seq_ids = prm->seq_ids;
    a.seen = prm->seen;
    a.weights = prm->weights;
    a.positions = prm->positions;
    a.weight_stride = prm->weight_stride;
    a.out_stride = prm->out_stride;
    a.kept = prm->kept;
    a.weights_out = prm->weights_out;
    a.positions_out = prm->positions_out;
    a.max_len = (int32_t)std::min<int64_t>((int64_t)c.max_blocks_per_seq * c.block_tokens, EKV_MAX_EVICT_TOKENS);
    return ekv::launch_evict(a, max_len, (cudaStream_t)stream);
}

int ekv_compact(ekv_pool *p, const ekv_compact_params *prm, ekv_stream_t stream) {
    if (!p || !prm || !prm->seq_ids || !prm->n_keep || !prm->slots) return EKV_ERR_INVALID_ARG;
    const ekv_pool_config &c = p->cfg;
    if (prm->layer0 < 0 || prm->n_layers <= 0 || prm->n_layers > c.n_layers - prm->layer0 || prm->n_batch < 0 || prm->slot_stride < 0)
        return EKV_ERR_INVALID_ARG;
    if (((uintptr_t)prm->seq_ids | (uintptr_t)prm->n_keep | (uintptr_t)prm->slots) & 3) return EKV_ERR_INVALID_ARG;
    if (prm->n_batch == 0 || prm->slot_stride == 0) return EKV_OK;
    const DeviceScope dev_scope(p);
    if (const int e = dev_scope.rc()) return e;
    ekv::CompactArgs a{};
    a.pool = p->view;
    a.layer0 = prm->layer0;
    a.n_layers = prm->n_layers;
    a.n_batch = prm->n_batch;
    a.seq_ids = prm->seq_ids;
    a.n_keep = prm->n_keep;
    a.slots = prm->slots;
    a.slot_stride = prm->slot_stride;
    return ekv::launch_compact(a, p->sms, (cudaStream_t)stream);
}

}  // extern "C"
