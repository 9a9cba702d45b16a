"""Python binding of libekv.so, the B200 paged KV-cache + masked-attention library.

A thin ctypes mirror of include/ekv.h for tests, the benchmark and Python callers: the pool
(`Pool`), sequence/block-table management, append / gather, and attention. Device buffers are
torch CUDA tensors (passed by data pointer); every call is asynchronous on the given (or
current) torch stream, like the C-ABI.

There is no fallback: if libekv.so is missing or fails to load, importing this module raises.
"""
from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass

HERE = os.path.dirname(os.path.abspath(__file__))
# EKV_LIB_PATH selects another build of the same library (e.g. a tracing build).
LIB_PATH = os.environ.get("EKV_LIB_PATH") or os.path.join(HERE, "libekv.so")

OK = 0
ERR_INVALID_ARG, ERR_CUDA, ERR_POOL_EXHAUSTED, ERR_NO_SEQ = -1, -2, -3, -4
ERR_RANGE, ERR_UNSUPPORTED, ERR_DEVICE, ERR_TIMEOUT, ERR_ALLOC = -5, -6, -7, -8, -9

DTYPE_F32, DTYPE_F16, DTYPE_Q8_0, DTYPE_BF16 = 0, 1, 8, 30
GATHER_NATIVE, GATHER_F32 = 0, 1
MASK_SUFFIX_CAUSAL = 1 << 0
MASK_SUFFIX_PREFIX_LM = 1 << 1
MASK_SPAN_ONLY = 1 << 2
MASK_SPAN_EXCLUDE = 1 << 3
MASK_BLOCK_CAUSAL = 1 << 4
MASK_FLEX_SELF = 1 << 5
MASK_FLEX_CROSS = 1 << 6


def flex_meta_word(seq: int, frame: int, clean: bool) -> int:
    """EKV_FLEX_META: the metadata word of a token for the FLEX masks (negative seq = padding)."""
    if seq < 0:
        return 0
    w = ((seq + 1) << 24) | ((1 if clean else 0) << 23) | (frame & 0x7FFFFF)
    return w - (1 << 32) if w >= (1 << 31) else w
ALGO_TC, ALGO_SIMT, ALGO_TC_PAIR, ALGO_TC_CTA, ALGO_TC_PAIR64, ALGO_TC_HEADS = 0, 1, 2, 3, 4, 5

# Device-side error codes written into the pool status word by kernels.
DEV_ERR_BAD_BLOCK, DEV_ERR_BAD_SEQ, DEV_ERR_BAD_POS, DEV_ERR_TIMEOUT, DEV_ERR_F16_RANGE = 1, 2, 3, 4, 5


class PoolConfig(C.Structure):
    _fields_ = [("device", C.c_int32), ("dtype", C.c_int32), ("block_tokens", C.c_int32),
                ("n_blocks", C.c_int32), ("kv_heads", C.c_int32), ("head_dim", C.c_int32),
                ("n_layers", C.c_int32), ("max_seqs", C.c_int32), ("max_blocks_per_seq", C.c_int32),
                ("suffix_tokens", C.c_int32)]


class PoolInfo(C.Structure):
    _fields_ = [("bytes_total", C.c_size_t), ("bytes_prefix", C.c_size_t),
                ("bytes_suffix", C.c_size_t), ("block_bytes", C.c_size_t),
                ("free_blocks", C.c_int32), ("live_seqs", C.c_int32),
                ("prefix_base", C.c_void_p), ("suffix_base", C.c_void_p),
                ("block_tables", C.c_void_p), ("seq_lens", C.c_void_p)]


class AttnParams(C.Structure):
    _fields_ = [("layer", C.c_int32), ("n_batch", C.c_int32), ("q_tokens", C.c_int32),
                ("q_heads", C.c_int32), ("scale", C.c_float), ("mask_flags", C.c_int32),
                ("chunk_tokens", C.c_int32), ("chunk_stride", C.c_int32),
                ("window_chunks", C.c_int32), ("q_chunk0", C.c_int32), ("suffix_len", C.c_int32),
                ("out_dtype", C.c_int32), ("use_prefix", C.c_int32), ("reserved", C.c_int32),
                ("seq_ids", C.c_void_p), ("prefix_len", C.c_void_p), ("prefix_valid", C.c_void_p),
                ("span_begin", C.c_void_p), ("span_end", C.c_void_p), ("flex_meta", C.c_void_p),
                ("flex_stride", C.c_int32), ("flex_q0", C.c_int32), ("flex_k0", C.c_int32),
                ("flex_window", C.c_int32)]


class SchedBatch(C.Structure):
    _fields_ = [("n_batch", C.c_int32), ("request_ids", C.POINTER(C.c_uint64)),
                ("seq_ids_host", C.POINTER(C.c_int32)), ("steps", C.POINTER(C.c_int32)),
                ("seq_ids", C.c_void_p), ("prefix_valid", C.c_void_p), ("n_admitted", C.c_int32),
                ("max_admitted_prefix", C.c_int32), ("admitted_index", C.POINTER(C.c_int32)),
                ("admitted_seq_ids", C.c_void_p), ("admitted_zeros", C.c_void_p),
                ("admitted_prefix_len", C.c_void_p), ("admitted_src_row", C.c_void_p), ("admitted_rows", C.c_int32),
                ("blocks_reused", C.c_int64), ("queued", C.c_int32)]


ROPE_HALF, ROPE_INTERLEAVED = 0, 1
MAX_DRAFT = 64
MAX_EVICT_TOKENS = 1 << 19


class RopeConfig(C.Structure):
    _fields_ = [("device", C.c_int32), ("layout", C.c_int32), ("rotary_dims", C.c_int32), ("n_ctx_orig", C.c_int32),
                ("freq_base", C.c_float), ("freq_scale", C.c_float), ("ext_factor", C.c_float),
                ("attn_factor", C.c_float), ("beta_fast", C.c_float), ("beta_slow", C.c_float),
                ("freq_factors", C.POINTER(C.c_float))]


class TreeParams(C.Structure):
    _fields_ = [("layer", C.c_int32), ("n_batch", C.c_int32), ("n_draft", C.c_int32), ("q_heads", C.c_int32),
                ("scale", C.c_float), ("softcap", C.c_float), ("out_dtype", C.c_int32), ("max_prefix", C.c_int32),
                ("seq_ids", C.c_void_p), ("prefix_len", C.c_void_p), ("n_nodes", C.c_void_p), ("ancestors", C.c_void_p)]


class EvictParams(C.Structure):
    _fields_ = [("layer0", C.c_int32), ("n_layers", C.c_int32), ("n_batch", C.c_int32), ("keep", C.c_int32),
                ("first", C.c_int32), ("recent", C.c_int32), ("seq_ids", C.c_void_p), ("seen", C.c_void_p),
                ("weights", C.c_void_p), ("positions", C.c_void_p), ("weight_stride", C.c_int64), ("kept", C.c_void_p),
                ("weights_out", C.c_void_p), ("positions_out", C.c_void_p), ("out_stride", C.c_int64)]


class CompactParams(C.Structure):
    _fields_ = [("layer0", C.c_int32), ("n_layers", C.c_int32), ("n_batch", C.c_int32), ("reserved", C.c_int32),
                ("seq_ids", C.c_void_p), ("n_keep", C.c_void_p), ("slots", C.c_void_p), ("slot_stride", C.c_int64)]


class WindowParams(C.Structure):
    _fields_ = [("layer", C.c_int32), ("n_batch", C.c_int32), ("q_heads", C.c_int32), ("max_rows", C.c_int32),
                ("window", C.c_int32), ("sinks", C.c_int32), ("scale", C.c_float), ("max_len", C.c_int32),
                ("seq_ids", C.c_void_p), ("dst_pos", C.c_void_p), ("n_rows", C.c_void_p), ("src_row", C.c_void_p)]


class HeadNormConfig(C.Structure):
    _fields_ = [("q_weight", C.c_void_p), ("k_weight", C.c_void_p), ("weight_dtype", C.c_int32),
                ("after_rotation", C.c_int32), ("weight_offset", C.c_float), ("eps", C.c_float)]


class Tensor(C.Structure):
    """ekv_tensor: a ggml-ordered strided device tensor (ne[0] fastest, nb in bytes)."""
    _fields_ = [("data", C.c_void_p), ("type", C.c_int32), ("ne", C.c_int64 * 4), ("nb", C.c_int64 * 4)]


# Every symbol include/ekv.h declares; tests check that the library exports all of them.
EXPORTED = [
    "ekv_pool_create", "ekv_pool_destroy", "ekv_pool_get_info", "ekv_pool_status", "ekv_pool_sync",
    "ekv_seq_create", "ekv_seq_free", "ekv_seq_resize", "ekv_seq_set_blocks", "ekv_seq_evict_front",
    "ekv_seq_append_tokens", "ekv_seq_clear_pred", "ekv_seq_restore", "ekv_seq_get_pred",
    "ekv_seq_get", "ekv_append", "ekv_append_suffix", "ekv_gather", "ekv_gather_suffix",
    "ekv_attention_workspace_size", "ekv_attention", "ekv_attention_algo", "ekv_version",
    "ekv_strerror", "ekv_attention_noalloc", "ekv_flash_attn_ext",
    "ekv_mul_mat_soft_max_mul_mat", "ekv_flash_attn_ext_workspace_size", "ekv_flash_attn_ext_ws",
    "ekv_mul_mat_soft_max_mul_mat_workspace_size", "ekv_mul_mat_soft_max_mul_mat_ws", "ekv_append_suffix_attention", "ekv_launch_count", "ekv_debug_expire_wait",
    "ekv_flow_step_f32", "ekv_guidance_f32", "ekv_sched_create", "ekv_sched_destroy", "ekv_sched_submit",
    "ekv_sched_begin_tick", "ekv_sched_end_tick", "ekv_sched_stats", "ekv_project_qkv_rope",
    "ekv_rope_create", "ekv_rope_destroy", "ekv_rope_get", "ekv_rope_append", "ekv_tree_attention_workspace_size",
    "ekv_tree_attention", "ekv_key_weights", "ekv_evict_by_weight", "ekv_norm_rope_append", "ekv_seq_drop_blocks",
    "ekv_seq_fork", "ekv_seq_own", "ekv_compact", "ekv_window_attention_workspace_size", "ekv_window_attention",
]
NOALLOC_SCRATCH_BYTES = 16 << 20  # EKV_NOALLOC_SCRATCH_BYTES


def _load():
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build it with `python embodied.cpp_b200/build.py`"
                          " (there is no CPU fallback)")
    L = C.CDLL(LIB_PATH)
    vp, i32, pi32 = C.c_void_p, C.c_int32, C.POINTER(C.c_int32)
    sig = {
        "ekv_pool_create": ([C.POINTER(PoolConfig), C.POINTER(vp)], C.c_int),
        "ekv_pool_destroy": ([vp], C.c_int),
        "ekv_pool_get_info": ([vp, C.POINTER(PoolInfo)], C.c_int),
        "ekv_pool_status": ([vp, pi32, vp], C.c_int),
        "ekv_pool_sync": ([vp, vp], C.c_int),
        "ekv_seq_create": ([vp, pi32], C.c_int),
        "ekv_seq_free": ([vp, i32], C.c_int),
        "ekv_seq_resize": ([vp, i32, i32], C.c_int),
        "ekv_seq_set_blocks": ([vp, i32, pi32, i32, i32], C.c_int),
        "ekv_seq_evict_front": ([vp, i32, i32], C.c_int),
        "ekv_seq_append_tokens": ([vp, i32, i32, i32], C.c_int),
        "ekv_seq_clear_pred": ([vp, i32], C.c_int),
        "ekv_debug_expire_wait": ([i32], C.c_int),
        "ekv_flow_step_f32": ([vp, vp, C.c_int64, C.c_float, i32, vp], C.c_int),
        "ekv_guidance_f32": ([vp, vp, C.c_int64, C.c_float, i32, i32, vp], C.c_int),
        "ekv_seq_restore": ([vp, i32, i32], C.c_int),
        "ekv_sched_create": ([vp, i32, i32, C.POINTER(vp)], C.c_int),
        "ekv_sched_destroy": ([vp], C.c_int),
        "ekv_sched_submit": ([vp, C.c_uint64, i32, i32], C.c_int),
        "ekv_sched_begin_tick": ([vp, C.POINTER(SchedBatch), vp], C.c_int),
        "ekv_sched_end_tick": ([vp, C.POINTER(C.c_uint64), i32, pi32], C.c_int),
        "ekv_sched_stats": ([vp, C.POINTER(C.c_int64), C.POINTER(C.c_int64), pi32, pi32], C.c_int),
        "ekv_seq_get_pred": ([vp, i32, pi32, pi32], C.c_int),
        "ekv_seq_get": ([vp, i32, pi32, pi32, pi32, i32], C.c_int),
        "ekv_append": ([vp, i32, i32, vp, vp, vp, vp, i32, vp, vp, vp], C.c_int),
        "ekv_append_suffix": ([vp, i32, i32, vp, i32, vp, vp, vp], C.c_int),
        "ekv_gather": ([vp, i32, i32, i32, i32, i32, vp, vp, vp], C.c_int),
        "ekv_gather_suffix": ([vp, i32, i32, i32, i32, vp, vp, vp], C.c_int),
        "ekv_attention_workspace_size": ([vp, C.POINTER(AttnParams)], C.c_size_t),
        "ekv_attention": ([vp, C.POINTER(AttnParams), vp, vp, vp, C.c_size_t, vp], C.c_int),
        "ekv_attention_algo": ([vp, C.POINTER(AttnParams), vp, vp, vp, C.c_size_t, i32, vp], C.c_int),
        "ekv_attention_noalloc": ([vp, C.POINTER(AttnParams), vp, vp, vp], C.c_int),
        "ekv_append_suffix_attention": ([vp, C.POINTER(AttnParams), vp, vp, vp, vp, vp, C.c_size_t, vp], C.c_int),
        "ekv_flash_attn_ext": ([C.POINTER(Tensor)] * 4 + [C.c_float] * 3 + [C.POINTER(Tensor), vp], C.c_int),
        "ekv_mul_mat_soft_max_mul_mat": ([C.POINTER(Tensor)] * 4 + [C.c_float] * 2 + [C.POINTER(Tensor), vp],
                                         C.c_int),
        "ekv_flash_attn_ext_workspace_size": ([C.POINTER(Tensor)] * 4 + [C.c_float] * 2 + [C.POINTER(Tensor)],
                                              C.c_size_t),
        "ekv_flash_attn_ext_ws": ([C.POINTER(Tensor)] * 4 + [C.c_float] * 3 + [C.POINTER(Tensor), vp, C.c_size_t, vp],
                                  C.c_int),
        "ekv_mul_mat_soft_max_mul_mat_workspace_size": ([C.POINTER(Tensor)] * 4 + [C.c_float, C.POINTER(Tensor)],
                                                        C.c_size_t),
        "ekv_mul_mat_soft_max_mul_mat_ws": ([C.POINTER(Tensor)] * 4 + [C.c_float] * 2 + [C.POINTER(Tensor), vp,
                                                                                         C.c_size_t, vp], C.c_int),
        "ekv_project_qkv_rope": ([vp, i32, i32, vp, i32, i32, i32, vp, vp, vp, vp, vp, C.c_float, vp, vp, vp, vp],
                                 C.c_int),
        "ekv_rope_create": ([C.POINTER(RopeConfig), C.POINTER(vp)], C.c_int),
        "ekv_rope_destroy": ([vp], C.c_int),
        "ekv_rope_get": ([vp, C.POINTER(C.c_double), i32, C.POINTER(C.c_float)], C.c_int),
        "ekv_rope_append": ([vp, vp, i32, i32, vp, vp, vp, vp, i32, vp, i32, vp, C.c_int64, vp, vp, vp, C.c_int64, vp],
                            C.c_int),
        "ekv_tree_attention_workspace_size": ([vp, C.POINTER(TreeParams)], C.c_size_t),
        "ekv_tree_attention": ([vp, C.POINTER(TreeParams), vp, vp, vp, vp, vp, vp, C.c_size_t, vp], C.c_int),
        "ekv_key_weights": ([vp, C.POINTER(TreeParams), vp, vp, vp, C.c_int64, C.c_float, vp], C.c_int),
        "ekv_evict_by_weight": ([vp, C.POINTER(EvictParams), vp], C.c_int),
        "ekv_norm_rope_append": ([vp, vp, C.POINTER(HeadNormConfig), i32, i32, vp, vp, vp, vp, i32, vp, i32, vp, C.c_int64, vp, vp,
                                  vp, C.c_int64, vp], C.c_int),
        "ekv_window_attention_workspace_size": ([vp, C.POINTER(WindowParams)], C.c_size_t),
        "ekv_window_attention": ([vp, C.POINTER(WindowParams), vp, C.c_int64, vp, vp, C.c_size_t, vp], C.c_int),
        "ekv_seq_drop_blocks": ([vp, i32, i32, i32], C.c_int),
        "ekv_seq_fork": ([vp, i32, pi32, pi32, pi32, vp], C.c_int),
        "ekv_seq_own": ([vp, i32, i32, i32, vp], C.c_int),
        "ekv_compact": ([vp, C.POINTER(CompactParams), vp], C.c_int),
        "ekv_version": ([], C.c_char_p),
        "ekv_launch_count": ([], C.c_uint64),
        "ekv_strerror": ([C.c_int], C.c_char_p),
    }
    for name, (args, res) in sig.items():
        f = getattr(L, name)
        f.argtypes = args
        f.restype = res
    return L


lib = _load()


class EkvError(RuntimeError):
    def __init__(self, code, what):
        super().__init__(f"{what}: {lib.ekv_strerror(code).decode()} ({code})")
        self.code = code


def check(code, what="ekv"):
    if code != OK:
        raise EkvError(code, what)
    return code


def _ptr(t):
    return None if t is None else t.data_ptr()


_bf16 = _f32 = _i32 = None  # torch's types, once a call has met a tensor


def _check_rows(*rows):
    """(tensor, elements, f32?, name) each: raises unless the tensor holds that many adjacent elements of bf16 (or of its
    bits) or f32. The calls ask for the usual case in line first: this takes 2 us of a call that may itself take 9."""
    global _bf16, _f32, _i32
    import torch
    _bf16, _f32, _i32 = torch.bfloat16, torch.float32, torch.int32
    for t, n, f32, name in rows:
        types = (_f32,) if f32 else (_bf16, torch.int16, torch.uint16)
        if t is not None and not (t.is_contiguous() and t.numel() >= n and t.dtype in types):
            raise ValueError(f"{name} must be {n} adjacent {'f32' if f32 else 'bf16'} values or more, in one piece")


def _index(t, n, name, bits=32):
    """The pointer of an integer array (a tensor, or a DevArray of the library) of at least n elements."""
    if t is None:
        return None
    if t.numel() < n or (hasattr(t, "is_contiguous") and not (t.is_contiguous() and t.dtype in _ints(bits))):
        raise ValueError(f"{name} must be {n} adjacent {bits}-bit integers or more, in one piece")
    return t.data_ptr()


def _rope_index(seq_ids, dst_pos, n_rows, src_row, positions, rows, append):
    """Requests of a rotary append and the pointers of its arrays: 32-bit integers, one for each request, positions for each of
    `rows` rows. (As _index asks, but the usual case in line: five calls of it take 3 us of one that takes 9, this 1.)"""
    global _i32
    n, i32 = n_rows.numel(), _i32
    try:
        # (of one element there is no distance to the next)
        if (n_rows.dtype is i32 and src_row.dtype is i32 and positions.dtype is i32 and src_row.numel() >= n and positions.numel() >= rows
                and (n == 1 or n_rows.is_contiguous() and src_row.is_contiguous()) and (rows == 1 or positions.is_contiguous())):
            if not append:
                return n, None, None, n_rows.data_ptr(), src_row.data_ptr(), positions.data_ptr()
            if (seq_ids.dtype is i32 and dst_pos.dtype is i32 and seq_ids.numel() >= n and dst_pos.numel() >= n
                    and (n == 1 or seq_ids.is_contiguous() and dst_pos.is_contiguous())):
                return n, seq_ids.data_ptr(), dst_pos.data_ptr(), n_rows.data_ptr(), src_row.data_ptr(), positions.data_ptr()
    except AttributeError:  # (an array of the library, or none: the call refuses it)
        pass
    _i32 = _ints(32)[0]
    return (n, _index(seq_ids, n, "seq_ids") if append else None, _index(dst_pos, n, "dst_pos") if append else None,
            _index(n_rows, n, "n_rows"), _index(src_row, n, "src_row"), _index(positions, rows, "positions"))


def _ints(bits):
    import torch
    return (torch.int32, torch.uint32) if bits == 32 else (torch.int64, torch.uint64)


def _current_stream():
    """The current torch stream's handle. torch.cuda.current_stream() makes a Stream object first, 3 us of a call that
    may itself take 5; where torch has the raw query it is asked instead."""
    global _current_stream
    import torch
    raw, device = getattr(torch._C, "_cuda_getCurrentRawStream", None), torch.cuda.current_device
    if raw is not None:
        _current_stream = lambda: raw(device())  # noqa: E731
    else:
        _current_stream = lambda: torch.cuda.current_stream().cuda_stream  # noqa: E731
    return _current_stream()


def _stream(stream):
    return _current_stream() if stream is None else stream.cuda_stream


@dataclass
class SeqView:
    n_tokens: int
    blocks: list


class Pool:
    """A paged KV pool on one device (ekv_pool_create / ekv_pool_destroy)."""

    def __init__(self, *, device=0, dtype=DTYPE_BF16, block_tokens=16, n_blocks=1024, kv_heads=1,
                 head_dim=256, n_layers=1, max_seqs=64, max_blocks_per_seq=64, suffix_tokens=0):
        self.cfg = PoolConfig(device, dtype, block_tokens, n_blocks, kv_heads, head_dim, n_layers,
                              max_seqs, max_blocks_per_seq, suffix_tokens)
        h = C.c_void_p()
        check(lib.ekv_pool_create(C.byref(self.cfg), C.byref(h)), "ekv_pool_create")
        self.h = h
        self.head_dim, self.kv_heads = head_dim, kv_heads  # (a field of cfg takes as long as a small check)

    def close(self):
        if self.h:
            check(lib.ekv_pool_destroy(self.h), "ekv_pool_destroy")
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def info(self) -> PoolInfo:
        i = PoolInfo()
        check(lib.ekv_pool_get_info(self.h, C.byref(i)), "ekv_pool_get_info")
        return i

    def status(self, stream=None) -> int:
        code = C.c_int32()
        check(lib.ekv_pool_status(self.h, C.byref(code), _stream(stream)), "ekv_pool_status")
        return code.value

    def sync(self, stream=None):
        check(lib.ekv_pool_sync(self.h, _stream(stream)), "ekv_pool_sync")

    # ---- sequences ----
    def seq_create(self) -> int:
        s = C.c_int32()
        check(lib.ekv_seq_create(self.h, C.byref(s)), "ekv_seq_create")
        return s.value

    def seq_free(self, seq):
        code = lib.ekv_seq_free(self.h, seq)
        if code:
            check(code, "ekv_seq_free")

    def seq_resize(self, seq, n_tokens):
        check(lib.ekv_seq_resize(self.h, seq, n_tokens), "ekv_seq_resize")

    def seq_set_blocks(self, seq, blocks, n_tokens):
        arr = (C.c_int32 * len(blocks))(*blocks)
        check(lib.ekv_seq_set_blocks(self.h, seq, arr, len(blocks), n_tokens), "ekv_seq_set_blocks")

    def seq_evict_front(self, seq, n_blocks):
        check(lib.ekv_seq_evict_front(self.h, seq, n_blocks), "ekv_seq_evict_front")

    def seq_drop_blocks(self, seq, first, n_blocks):
        """ekv_seq_drop_blocks: blocks [first, first + n_blocks) leave the sequence; later tokens move down."""
        check(lib.ekv_seq_drop_blocks(self.h, seq, first, n_blocks), "ekv_seq_drop_blocks")

    def seq_fork(self, parents, n_tokens, stream=None) -> list:
        """ekv_seq_fork: one new sequence for each entry, the first n_tokens[i] tokens of sequence parents[i]; whole blocks
        are shared, the last, partial one is copied. Needs no sync()."""
        n = len(parents)
        if len(n_tokens) != n:
            raise ValueError("one length for each parent")
        ints = C.c_int32 * n
        children = ints()
        code = lib.ekv_seq_fork(self.h, n, ints(*parents), ints(*n_tokens), children,
                                None if self.cfg.device < 0 else _stream(stream))
        if code:
            check(code, "ekv_seq_fork")
        return children[:]

    def seq_own(self, seq, pos0, n_tokens, stream=None):
        """ekv_seq_own: shared blocks under positions [pos0, pos0 + n_tokens) become copies that the sequence may write."""
        check(lib.ekv_seq_own(self.h, seq, pos0, n_tokens, None if self.cfg.device < 0 else _stream(stream)), "ekv_seq_own")

    def seq_append_tokens(self, seq, n_tokens, pred=False):
        check(lib.ekv_seq_append_tokens(self.h, seq, n_tokens, 1 if pred else 0), "ekv_seq_append_tokens")

    def seq_clear_pred(self, seq):
        check(lib.ekv_seq_clear_pred(self.h, seq), "ekv_seq_clear_pred")

    def seq_restore(self, seq, n_tokens):
        check(lib.ekv_seq_restore(self.h, seq, n_tokens), "ekv_seq_restore")

    def seq_get_pred(self, seq):
        lo, hi = C.c_int32(), C.c_int32()
        check(lib.ekv_seq_get_pred(self.h, seq, C.byref(lo), C.byref(hi)), "ekv_seq_get_pred")
        return lo.value, hi.value

    def seq_get(self, seq) -> SeqView:
        nt, nb = C.c_int32(), C.c_int32()
        check(lib.ekv_seq_get(self.h, seq, C.byref(nt), C.byref(nb), None, 0), "ekv_seq_get")
        arr = (C.c_int32 * max(1, nb.value))()
        check(lib.ekv_seq_get(self.h, seq, None, None, arr, nb.value), "ekv_seq_get")
        return SeqView(nt.value, list(arr)[: nb.value])

    # ---- data ----
    def append(self, layer, seq_ids, dst_pos, n_rows, src_row, max_rows, k, v, stream=None):
        check(lib.ekv_append(self.h, layer, seq_ids.numel(), _ptr(seq_ids), _ptr(dst_pos),
                             _ptr(n_rows), _ptr(src_row), max_rows, _ptr(k), _ptr(v),
                             _stream(stream)), "ekv_append")

    def append_suffix(self, layer, seq_ids, k, v, stream=None):
        n_rows = k.shape[1]
        check(lib.ekv_append_suffix(self.h, layer, seq_ids.numel(), _ptr(seq_ids), n_rows, _ptr(k),
                                    _ptr(v), _stream(stream)), "ekv_append_suffix")

    def gather(self, layer, seq, pos0, n_rows, fmt, k_out, v_out, stream=None):
        check(lib.ekv_gather(self.h, layer, seq, pos0, n_rows, fmt, _ptr(k_out), _ptr(v_out),
                             _stream(stream)), "ekv_gather")

    def gather_suffix(self, layer, seq, n_rows, fmt, k_out, v_out, stream=None):
        check(lib.ekv_gather_suffix(self.h, layer, seq, n_rows, fmt, _ptr(k_out), _ptr(v_out),
                                    _stream(stream)), "ekv_gather_suffix")

    def attention_params(self, *, layer, seq_ids, q_tokens, q_heads, scale, mask_flags=0,
                         chunk_tokens=0, chunk_stride=0, window_chunks=0, q_chunk0=0,
                         suffix_len=0, out_dtype=DTYPE_BF16, use_prefix=True, prefix_len=None,
                         prefix_valid=None, span_begin=None, span_end=None, flex_meta=None, flex_stride=0,
                         flex_q0=0, flex_k0=0, flex_window=0) -> AttnParams:
        p = AttnParams(layer, seq_ids.numel(), q_tokens, q_heads, scale, mask_flags, chunk_tokens,
                       chunk_stride, window_chunks, q_chunk0, suffix_len, out_dtype,
                       1 if use_prefix else 0, 0, seq_ids.data_ptr(),
                       None if prefix_len is None else prefix_len.data_ptr(),
                       None if prefix_valid is None else prefix_valid.data_ptr(),
                       None if span_begin is None else span_begin.data_ptr(),
                       None if span_end is None else span_end.data_ptr(),
                       None if flex_meta is None else flex_meta.data_ptr(), flex_stride, flex_q0, flex_k0,
                       flex_window)
        p._keep = (seq_ids, prefix_len, prefix_valid, span_begin, span_end, flex_meta)
        return p

    def workspace_size(self, params: AttnParams) -> int:
        return lib.ekv_attention_workspace_size(self.h, C.byref(params))

    def attention(self, params: AttnParams, q, out, workspace=None, algo=ALGO_TC, stream=None):
        ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
        check(lib.ekv_attention_algo(self.h, C.byref(params), _ptr(q), _ptr(out), _ptr(workspace),
                                     ws_bytes, algo, _stream(stream)), "ekv_attention")

    def append_suffix_attention(self, params: AttnParams, k_suffix, v_suffix, q, out, workspace=None, stream=None):
        """ekv_append_suffix_attention: this layer-step's suffix K/V ([n_batch][suffix_len][kv_heads]
        [head_dim] bf16) into the slots, then attention, in one call."""
        ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
        check(lib.ekv_append_suffix_attention(self.h, C.byref(params), _ptr(k_suffix), _ptr(v_suffix), _ptr(q),
                                              _ptr(out), _ptr(workspace), ws_bytes, _stream(stream)),
              "ekv_append_suffix_attention")


    # ---- token-by-token decoding ----
    def rope_append(self, rope, layer, seq_ids, dst_pos, n_rows, src_row, max_rows, positions, *, q=None, q_out=None,
                    k=None, v=None, stream=None):
        """ekv_rope_append: turn q [rows, q_heads, head_dim] into q_out and k into the pages beside v ([rows, kv_heads,
        head_dim]), all bf16 and by source row. q, k and v may be slices of one [rows, columns] projection output:
        rows may be any distance apart, a row's heads are adjacent. Either pair may be left out."""
        _, q_heads, qp, q_stride, q_to, kp, vp, kv_stride = self._rope_rows(q, q_out, k, v)
        # (positions may end with the last row that a request uses, which only the device knows)
        n, seqs, dst, counts, src, pos = _rope_index(seq_ids, dst_pos, n_rows, src_row, positions, 0, kp is not None)
        code = lib.ekv_rope_append(self.h, rope.h, layer, n, seqs, dst, counts, src, max_rows, pos, q_heads, qp, q_stride, q_to, kp, vp,
                                   kv_stride, _stream(stream))
        if code:
            check(code, "ekv_rope_append")

    def _rope_rows(self, q, q_out, k, v):
        """Rows, heads, pointers and row distances of a rotary append. (Shapes and distances are asked for once: each takes 0.2 us.)"""
        rows = q_heads = q_stride = kv_stride = 0
        qp = q_to = kp = vp = None
        if q is not None:
            shape = q.shape
            rows = shape[0]
            q_heads, q_stride = _rows_of(shape, q.stride(), self.head_dim, "q")
            if q_out is None or q_out.shape != shape or not q_out.is_contiguous():
                raise ValueError("q_out must be contiguous and of q's shape")
            qp, q_to = q.data_ptr(), q_out.data_ptr()
        if k is not None or v is not None:
            if k is None or v is None:
                raise ValueError("k and v must have one shape and the same distance from row to row")
            shape, steps = k.shape, k.stride()
            if shape != v.shape or steps != v.stride():
                raise ValueError("k and v must have one shape and the same distance from row to row")
            kv_heads, kv_stride = _rows_of(shape, steps, self.head_dim, "k and v")
            if kv_heads != self.kv_heads:
                raise ValueError("k and v must have the pool's KV heads")
            kp, vp = k.data_ptr(), v.data_ptr()
            rows = max(rows, shape[0])
        return rows, q_heads, qp, q_stride, q_to, kp, vp, kv_stride

    def norm_rope_append(self, rope, norm, layer, seq_ids, dst_pos, n_rows, src_row, max_rows, positions, *, q=None, q_out=None,
                         k=None, v=None, stream=None):
        """ekv_norm_rope_append: rope_append with an RMS norm (HeadNorm) of every q and k head before its rotation, or after. positions
        has a value for every row of q and k."""
        if norm.dim not in (0, self.head_dim):
            raise ValueError("the norm's weights must have head_dim values")
        rows, q_heads, qp, q_stride, q_to, kp, vp, kv_stride = self._rope_rows(q, q_out, k, v)
        bf16 = norm.bf16
        if not ((qp is None or q.dtype is bf16 and q_out.dtype is bf16) and (kp is None or k.dtype is bf16 and v.dtype is bf16)):
            raise ValueError("q, q_out, k and v must be bf16")
        n, seqs, dst, counts, src, pos = _rope_index(seq_ids, dst_pos, n_rows, src_row, positions, rows, kp is not None)
        code = lib.ekv_norm_rope_append(self.h, rope.h, norm.ref, layer, n, seqs, dst, counts, src, max_rows, pos, q_heads, qp, q_stride,
                                        q_to, kp, vp, kv_stride, _stream(stream))
        if code:
            check(code, "ekv_norm_rope_append")

    def tree_params(self, *, layer, seq_ids, n_draft, q_heads, scale, softcap=0.0, out_dtype=DTYPE_BF16,
                    prefix_len=None, n_nodes=None, ancestors=None, max_prefix=0) -> TreeParams:
        """What ekv_tree_attention and ekv_key_weights share. max_prefix, the longest cached prefix of the call, is worth
        giving where the pool holds longer sequences that are not of the call."""
        n = seq_ids.numel()
        p = TreeParams(layer, n, n_draft, q_heads, scale, softcap, out_dtype, max_prefix, _index(seq_ids, n, "seq_ids"),
                       _index(prefix_len, n, "prefix_len"), _index(n_nodes, n, "n_nodes"),
                       _index(ancestors, n * n_draft, "ancestors", 64))
        p._keep = (seq_ids, prefix_len, n_nodes, ancestors)
        return p

    def tree_attention_workspace_size(self, params: TreeParams) -> int:
        return lib.ekv_tree_attention_workspace_size(self.h, C.byref(params))

    def tree_attention(self, params: TreeParams, q, k_draft, v_draft, out, lse=None, workspace=None, stream=None):
        """ekv_tree_attention: q [n_batch, n_draft, q_heads, head_dim], k_draft / v_draft [n_batch, n_draft, kv_heads,
        head_dim] bf16 over the cached prefix; out like q (bf16 or f32), lse f32 [n_batch, n_draft, q_heads]. All in one
        piece: a slice of a projection needs .contiguous() first."""
        rows, dim = params.n_batch * params.n_draft, self.head_dim
        heads = rows * params.q_heads
        n, m, f32 = heads * dim, rows * self.kv_heads * dim, params.out_dtype == DTYPE_F32
        bf16 = _bf16
        if not (q.dtype is bf16 and k_draft.dtype is bf16 and v_draft.dtype is bf16 and out.dtype is (_f32 if f32 else bf16)
                and q.is_contiguous() and k_draft.is_contiguous() and v_draft.is_contiguous() and out.is_contiguous()
                and q.numel() >= n and k_draft.numel() >= m and v_draft.numel() >= m and out.numel() >= n
                and (lse is None or lse.dtype is _f32 and lse.is_contiguous() and lse.numel() >= heads)):
            _check_rows((q, n, False, "q"), (k_draft, m, False, "k_draft"), (v_draft, m, False, "v_draft"), (out, n, f32, "out"),
                        (lse, heads, True, "lse"))
        ws_bytes = 0
        if workspace is not None:
            if not workspace.is_contiguous():
                raise ValueError("workspace must be in one piece")
            ws_bytes = workspace.numel() * workspace.element_size()
        code = lib.ekv_tree_attention(self.h, C.byref(params), q.data_ptr(), k_draft.data_ptr(), v_draft.data_ptr(),
                                      out.data_ptr(), _ptr(lse), _ptr(workspace), ws_bytes, _stream(stream))
        if code:
            check(code, "ekv_tree_attention")

    def key_weights(self, params: TreeParams, q, lse, weights, decay=1.0, stream=None):
        """ekv_key_weights: weights [n_batch, kv_heads, stride] f32 = decay * weights + what the rows give each key; q and
        lse as ekv_tree_attention got and gave them."""
        heads, stride = params.n_batch * params.n_draft * params.q_heads, weights.shape[-1]
        n, m = heads * self.head_dim, params.n_batch * self.kv_heads * stride
        if not (q.dtype is _bf16 and lse.dtype is _f32 and weights.dtype is _f32 and q.is_contiguous() and lse.is_contiguous()
                and weights.is_contiguous() and q.numel() >= n and lse.numel() >= heads and weights.numel() >= m):
            _check_rows((q, n, False, "q"), (lse, heads, True, "lse"), (weights, m, True, "weights"))
        code = lib.ekv_key_weights(self.h, C.byref(params), q.data_ptr(), lse.data_ptr(), weights.data_ptr(), stride, decay,
                                   _stream(stream))
        if code:
            check(code, "ekv_key_weights")

    def evict_by_weight(self, layer0, n_layers, seq_ids, weights, *, keep, first, recent, kept, weights_out=None,
                        positions=None, positions_out=None, seen=None, stream=None):
        """ekv_evict_by_weight: weights (and positions) [n_layers, n_batch, kv_heads, stride], kept int32 [n_layers,
        n_batch, kv_heads, keep]; weights_out and positions_out have one stride of their own, or are the inputs."""
        n, stride = seq_ids.numel(), weights.shape[-1]
        rows, out_stride = n_layers * n * self.kv_heads, 0
        if weights_out is not None:
            out_stride = weights_out.shape[-1]
        elif positions_out is not None:
            out_stride = positions_out.shape[-1]
        if (positions_out is not None and positions_out.shape[-1] != out_stride
                or positions is not None and positions.shape[-1] != stride):
            raise ValueError("weights and positions have one stride, and so have the outputs")
        if kept.shape[-1] != keep and kept.dim() > 1:
            raise ValueError("kept must be [n_layers, n_batch, kv_heads, keep]")
        m, i32, f32 = rows * out_stride, _i32, _f32
        if not (kept.dtype is i32 and kept.is_contiguous() and kept.numel() >= rows * keep
                and (seq_ids.__class__ is DevArray or seq_ids.dtype is i32 and seq_ids.is_contiguous())
                and weights.dtype is f32 and weights.is_contiguous() and weights.numel() >= rows * stride
                and (weights_out is None or weights_out.dtype is f32 and weights_out.is_contiguous() and weights_out.numel() >= m)
                and (positions is None or positions.dtype is i32 and positions.is_contiguous() and positions.numel() >= rows * stride)
                and (positions_out is None or positions_out.dtype is i32 and positions_out.is_contiguous() and positions_out.numel() >= m)
                and (seen is None or seen.__class__ is not DevArray and seen.dtype is i32 and seen.is_contiguous() and seen.numel() >= n)):
            _check_rows((weights, rows * stride, True, "weights"), (weights_out, m, True, "weights_out"))
            for t, size, name in ((kept, rows * keep, "kept"), (positions, rows * stride, "positions"),
                                  (positions_out, m, "positions_out"), (seen, n, "seen"), (seq_ids, n, "seq_ids")):
                _index(t, size, name)
        p = EvictParams(layer0, n_layers, n, keep, first, recent, seq_ids.data_ptr(), None if seen is None else seen.data_ptr(),
                        weights.data_ptr(), None if positions is None else positions.data_ptr(), stride, kept.data_ptr(),
                        None if weights_out is None else weights_out.data_ptr(),
                        None if positions_out is None else positions_out.data_ptr(), out_stride)
        code = lib.ekv_evict_by_weight(self.h, C.byref(p), _stream(stream))
        if code:
            check(code, "ekv_evict_by_weight")


    def window_params(self, *, layer, seq_ids, dst_pos, n_rows, src_row, max_rows, q_heads, scale, window=0, sinks=0,
                      max_len=0) -> WindowParams:
        """What ekv_window_attention is asked: rows as ekv_append's (dst_pos, n_rows, src_row), a window (0: none) and the number
        of first slots that stay visible. max_len, the longest sequence of the call, is worth giving where the pool holds longer
        ones that are not of the call."""
        n = seq_ids.numel()
        p = WindowParams(layer, n, q_heads, max_rows, window, sinks, scale, max_len, _index(seq_ids, n, "seq_ids"),
                         _index(dst_pos, n, "dst_pos"), _index(n_rows, n, "n_rows"), _index(src_row, n, "src_row"))
        p._keep = (seq_ids, dst_pos, n_rows, src_row)
        p.heads = q_heads
        return p

    def window_attention_workspace_size(self, params: WindowParams) -> int:
        return lib.ekv_window_attention_workspace_size(self.h, C.byref(params))

    def window_attention(self, params: WindowParams, q, out, workspace=None, stream=None):
        """ekv_window_attention: q bf16 [rows, q_heads, head_dim], its rows any distance apart (a slice of a projection), out
        bf16 of q's shape, in one piece."""
        heads, stride = _rows(q, self.head_dim, "q")
        if heads != params.heads or q.dtype is not out.dtype or not out.is_contiguous() or out.shape != q.shape:
            raise ValueError("q must have params' query heads, and out must be contiguous and of q's shape and type")
        if q.dtype is not _bf16:
            import torch
            if q.dtype is not torch.bfloat16:
                raise ValueError("q and out must be bf16")
        ws_bytes = 0
        if workspace is not None:
            if not workspace.is_contiguous():
                raise ValueError("workspace must be in one piece")
            ws_bytes = workspace.numel() * workspace.element_size()
        code = lib.ekv_window_attention(self.h, C.byref(params), q.data_ptr(), stride, out.data_ptr(), _ptr(workspace), ws_bytes,
                                        _stream(stream))
        if code:
            check(code, "ekv_window_attention")

    def compact(self, layer0, n_layers, seq_ids, slots, n_keep, stream=None):
        """ekv_compact: slot i of sequence seq_ids[b] gets the row of slot slots[b, i], for i below n_keep[b], in the layers from
        layer0 on. slots int32 [n_batch, stride], ascending; call seq_resize(seq, n_keep) afterwards."""
        n = seq_ids.numel()
        if slots.dim() != 2 or slots.shape[0] != n:
            raise ValueError("slots must be [n_batch, stride]")
        stride = slots.shape[1]
        p = CompactParams(layer0, n_layers, n, 0, _index(seq_ids, n, "seq_ids"), _index(n_keep, n, "n_keep"),
                          _index(slots, n * stride, "slots"), stride)
        code = lib.ekv_compact(self.h, C.byref(p), _stream(stream))
        if code:
            check(code, "ekv_compact")


class HeadNorm:
    """RMS norms of q and k heads for norm_rope_append (ekv_head_norm): weights of head_dim values, bf16 or f32 (None: ones),
    weight_offset added to them (1 where they are stored as differences from 1), before the rotation or after it."""

    def __init__(self, *, q_weight=None, k_weight=None, eps=1e-6, weight_offset=0.0, after_rotation=False):
        import torch
        given = [w for w in (q_weight, k_weight) if w is not None]
        for w in given:
            if w.dtype not in (torch.float32, torch.bfloat16) or w.dim() != 1 or not w.is_contiguous():
                raise ValueError("weights must be one adjacent row of bf16 or f32 values")
        if len({(w.dtype, w.numel()) for w in given}) > 1:
            raise ValueError("q_weight and k_weight must have one type and length")
        self.dim = given[0].numel() if given else 0
        self.bf16 = torch.bfloat16
        self._keep = given
        self.cfg = HeadNormConfig(_ptr(q_weight), _ptr(k_weight),
                                  DTYPE_BF16 if given and given[0].dtype is torch.bfloat16 else DTYPE_F32,
                                  1 if after_rotation else 0, weight_offset, eps)
        self.ref = C.byref(self.cfg)


class Rope:
    """Rotary frequencies (ekv_rope_create): layout, rotated columns and long-context scaling, as ggml_rope_ext."""

    def __init__(self, *, device=0, interleaved=False, rotary_dims, freq_base=10000.0, freq_scale=1.0, ext_factor=0.0,
                 attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, n_ctx_orig=0, freq_factors=None):
        ff = None
        if freq_factors is not None:
            if len(freq_factors) != rotary_dims // 2:
                raise ValueError("freq_factors: one for each pair")
            ff = (C.c_float * len(freq_factors))(*freq_factors)
        cfg = RopeConfig(device, ROPE_INTERLEAVED if interleaved else ROPE_HALF, rotary_dims, n_ctx_orig, freq_base,
                         freq_scale, ext_factor, attn_factor, beta_fast, beta_slow, ff)
        self.rotary_dims = rotary_dims
        self.h = C.c_void_p()
        check(lib.ekv_rope_create(C.byref(cfg), C.byref(self.h)), "ekv_rope_create")

    def frequencies(self):
        """Radians per position of each pair, and the factor of the rotation."""
        f, m = (C.c_double * (self.rotary_dims // 2))(), C.c_float()
        check(lib.ekv_rope_get(self.h, f, self.rotary_dims // 2, C.byref(m)), "ekv_rope_get")
        return list(f), m.value

    def close(self):
        if self.h:
            check(lib.ekv_rope_destroy(self.h), "ekv_rope_destroy")
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def project_qkv_rope(pool: "Pool", layer, seq_ids, x, wq, wk, wv, positions, rope_base, q_out, k_out=None, v_out=None,
                     *, tokens, q_heads, stream=None):
    """ekv_project_qkv_rope: x [n_batch * tokens, hidden] bf16, weights [out, hidden] bf16, positions int32
    [n_batch * tokens]; q_out [n_batch, tokens, q_heads, head_dim] bf16; K/V into the pool's suffix slots
    (k_out / v_out None) or into k_out / v_out [n_batch, tokens, kv_heads, head_dim] bf16."""
    rows, hidden = x.shape
    n_batch = rows // tokens
    check(lib.ekv_project_qkv_rope(pool.h, layer, n_batch, _ptr(seq_ids), tokens, q_heads, hidden, _ptr(x), _ptr(wq),
                                   _ptr(wk), _ptr(wv), _ptr(positions), rope_base, _ptr(q_out), _ptr(k_out),
                                   _ptr(v_out), _stream(stream)), "ekv_project_qkv_rope")


def _rows(t, head_dim, name):
    """Heads of a [rows, heads, head_dim] tensor and the elements from row to row; a row must be adjacent."""
    return _rows_of(t.shape, t.stride(), head_dim, name)


def _rows_of(shape, steps, head_dim, name):
    if len(shape) == 3:
        rows, heads, dim = shape
        to_row, to_head, to_col = steps
        if dim == head_dim and to_col == 1 and (to_head == dim or heads <= 1):
            return heads, to_row if rows > 1 else heads * dim
    raise ValueError(f"{name} must be [rows, heads, {head_dim}] with adjacent heads")


class DevArray:
    """A device (or, for a host-only pool, host) int32 array owned by the library: what
    Pool.attention_params and Pool.append read from a tensor (numel, data_ptr)."""

    def __init__(self, ptr, n):
        self.ptr, self.n = ptr or 0, n

    def numel(self):
        return self.n

    def data_ptr(self):
        return self.ptr


@dataclass
class Tick:
    """One tick of the scheduler (ekv_sched_batch): every active request runs its next denoise step."""
    n_batch: int
    request_ids: list
    seq_ids_host: list
    steps: list
    seq_ids: DevArray
    prefix_valid: DevArray
    admitted_index: list
    admitted_seq_ids: DevArray
    admitted_zeros: DevArray
    admitted_prefix_len: DevArray
    admitted_src_row: DevArray
    admitted_rows: int
    max_admitted_prefix: int
    blocks_reused: int
    queued: int


class Scheduler:
    """Batching scheduler over a pool (ekv_sched_*): first come first served admission, one denoise
    step of every active request per tick, blocks freed (and reused) on completion."""

    def __init__(self, pool: Pool, max_batch: int, n_steps: int):
        self.pool = pool
        self.h = C.c_void_p()
        check(lib.ekv_sched_create(pool.h, max_batch, n_steps, C.byref(self.h)), "ekv_sched_create")

    def close(self):
        if self.h:
            lib.ekv_sched_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def submit(self, request_id, prefix_len, prefix_valid=None):
        pv = prefix_len if prefix_valid is None else prefix_valid
        check(lib.ekv_sched_submit(self.h, request_id, prefix_len, pv), "ekv_sched_submit")

    def begin_tick(self, stream=None) -> Tick:
        b = SchedBatch()
        s = None if self.pool.cfg.device < 0 else _stream(stream)
        check(lib.ekv_sched_begin_tick(self.h, C.byref(b), s), "ekv_sched_begin_tick")
        n, na = b.n_batch, b.n_admitted
        return Tick(n, list(b.request_ids[:n]) if n else [], list(b.seq_ids_host[:n]) if n else [],
                    list(b.steps[:n]) if n else [], DevArray(b.seq_ids, n), DevArray(b.prefix_valid, n),
                    list(b.admitted_index[:na]) if na else [], DevArray(b.admitted_seq_ids, na),
                    DevArray(b.admitted_zeros, na), DevArray(b.admitted_prefix_len, na),
                    DevArray(b.admitted_src_row, na), b.admitted_rows, b.max_admitted_prefix,
                    b.blocks_reused, b.queued)

    def end_tick(self, cap=4096) -> list:
        arr = (C.c_uint64 * cap)()
        nf = C.c_int32()
        check(lib.ekv_sched_end_tick(self.h, arr, cap, C.byref(nf)), "ekv_sched_end_tick")
        return list(arr[: min(nf.value, cap)])

    def stats(self) -> dict:
        c, r, a, q = C.c_int64(), C.c_int64(), C.c_int32(), C.c_int32()
        check(lib.ekv_sched_stats(self.h, C.byref(c), C.byref(r), C.byref(a), C.byref(q)), "ekv_sched_stats")
        return dict(completed=c.value, blocks_reused=r.value, active=a.value, queued=q.value)


def flow_step(sample, velocity, delta, bf16_round=False, stream=None):
    """ekv_flow_step_f32 on contiguous f32 torch tensors of equal size (sample updated in place)."""
    check(lib.ekv_flow_step_f32(_ptr(sample), _ptr(velocity), sample.numel(), float(delta), 1 if bf16_round else 0,
                                _stream(stream)), "ekv_flow_step_f32")


def guidance(cond, uncond, scale, use_guidance=True, bf16_round=False, stream=None):
    """ekv_guidance_f32 on contiguous f32 torch tensors (cond updated in place)."""
    check(lib.ekv_guidance_f32(_ptr(cond), _ptr(uncond), cond.numel(), float(scale), 1 if use_guidance else 0,
                               1 if bf16_round else 0, _stream(stream)), "ekv_guidance_f32")


_TORCH_DTYPES = {"torch.float32": DTYPE_F32, "torch.float16": DTYPE_F16, "torch.bfloat16": DTYPE_BF16}


def ggml_view(t) -> Tensor:
    """Describe a torch tensor (up to 4-D, any strides) as ekv_tensor in ggml order: the torch shape
    reversed, so a [B, H, T, D] tensor is ne = {D, T, H, B} and nb = its strides in bytes."""
    if t.dim() > 4:
        raise ValueError("at most 4 dimensions")
    dt = _TORCH_DTYPES.get(str(t.dtype))
    if dt is None:
        raise ValueError(f"unsupported dtype {t.dtype}")
    shape = [1] * (4 - t.dim()) + list(t.shape)
    strides = [0] * (4 - t.dim()) + list(t.stride())
    es = t.element_size()
    g = Tensor()
    g.data = t.data_ptr()
    g.type = dt
    for i in range(4):
        g.ne[i] = shape[3 - i]
        g.nb[i] = strides[3 - i] * es
    return g


def flash_attn_ext(q, k, v, mask, dst, *, scale, max_bias=0.0, logit_softcap=0.0, workspace=None, stream=None):
    """ggml_flash_attn_ext on torch tensors given in reversed ggml order: q [B, Hq, Tq, D],
    k [Bk, Hkv, Tk, D], v [Bk, Hkv, Tk, Dv], mask [Mb, Mh, >=Tq, >=Tk] (or None) and the f32
    result dst [B, Tq, Hq, Dv]; any of them may be a permuted or sliced view. With `workspace` (a
    uint8 device tensor of flash_attn_ext_workspace_size bytes) the call stages into it
    (ekv_flash_attn_ext_ws), else into the library's per-device workspace."""
    gm = None if mask is None else C.byref(ggml_view(mask))
    args = (C.byref(ggml_view(q)), C.byref(ggml_view(k)), C.byref(ggml_view(v)), gm, scale, max_bias, logit_softcap,
            C.byref(ggml_view(dst)))
    if workspace is None:
        check(lib.ekv_flash_attn_ext(*args, _stream(stream)), "ekv_flash_attn_ext")
    else:
        check(lib.ekv_flash_attn_ext_ws(*args, _ptr(workspace), workspace.numel() * workspace.element_size(),
                                        _stream(stream)), "ekv_flash_attn_ext_ws")


def flash_attn_ext_workspace_size(q, k, v, mask, dst, *, max_bias=0.0, logit_softcap=0.0) -> int:
    """Bytes of the tensor-core staging of this flash_attn_ext call (0: it runs on the CUDA cores)."""
    gm = None if mask is None else C.byref(ggml_view(mask))
    return lib.ekv_flash_attn_ext_workspace_size(C.byref(ggml_view(q)), C.byref(ggml_view(k)), C.byref(ggml_view(v)),
                                                 gm, max_bias, logit_softcap, C.byref(ggml_view(dst)))


def mul_mat_soft_max_mul_mat(k, q, v, mask, dst, *, scale, max_bias=0.0, workspace=None, stream=None):
    """The ggml triple mul_mat(K, Q) -> soft_max_ext -> mul_mat(V, .) on torch tensors in reversed ggml
    order: k [Bk, Hkv, Tk, D], q [B, Hq, Tq, D], v [Bk, Hkv, Dv, Tk] (keys fastest), mask
    [Mb, Mh, >=Tq, >=Tk] or None, f32 dst [B, Hq, Tq, Dv]. `workspace` as for flash_attn_ext."""
    gm = None if mask is None else C.byref(ggml_view(mask))
    args = (C.byref(ggml_view(k)), C.byref(ggml_view(q)), C.byref(ggml_view(v)), gm, scale, max_bias,
            C.byref(ggml_view(dst)))
    if workspace is None:
        check(lib.ekv_mul_mat_soft_max_mul_mat(*args, _stream(stream)), "ekv_mul_mat_soft_max_mul_mat")
    else:
        check(lib.ekv_mul_mat_soft_max_mul_mat_ws(*args, _ptr(workspace), workspace.numel() * workspace.element_size(),
                                                  _stream(stream)), "ekv_mul_mat_soft_max_mul_mat_ws")


def mul_mat_soft_max_mul_mat_workspace_size(k, q, v, mask, dst, *, max_bias=0.0) -> int:
    gm = None if mask is None else C.byref(ggml_view(mask))
    return lib.ekv_mul_mat_soft_max_mul_mat_workspace_size(C.byref(ggml_view(k)), C.byref(ggml_view(q)),
                                                           C.byref(ggml_view(v)), gm, max_bias,
                                                           C.byref(ggml_view(dst)))


def version() -> str:
    return lib.ekv_version().decode()
