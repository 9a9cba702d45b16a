"""Argument checks of the windowed attention; no kernel is launched (the pool is host-only, so a call that passes the checks ends with
EKV_ERR_UNSUPPORTED)."""
import ctypes as C
import math

import pytest
import torch

import ekv

P = 0x10000  # a pointer that is never followed
L = ekv.lib


def pool(**kw):
    cfg = dict(device=-1, dtype=ekv.DTYPE_BF16, block_tokens=16, n_blocks=40, kv_heads=2, head_dim=64, n_layers=2, max_seqs=6,
               max_blocks_per_seq=12)
    cfg.update(kw)
    return ekv.Pool(**cfg)


def params(**kw):
    p = ekv.WindowParams(0, 3, 8, 5, 100, 4, 0.125, 0, P, P, P, P)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def call(p, prm, q=P, stride=0, out=2 * P, ws=P):
    return L.ekv_window_attention(p.h, C.byref(prm), q, stride, out, ws, 1 << 20, None)


def test_refusals():
    p = pool()
    assert call(p, params()) == ekv.ERR_UNSUPPORTED  # no device
    for kw in (dict(layer=2), dict(layer=-1), dict(n_batch=-1), dict(max_rows=-1), dict(q_heads=0), dict(q_heads=7), dict(q_heads=-2),
               dict(window=-1), dict(sinks=-1), dict(max_len=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
               dict(scale=3e38), dict(seq_ids=None), dict(dst_pos=None), dict(n_rows=None), dict(src_row=None), dict(seq_ids=P + 2),
               dict(dst_pos=P + 1), dict(n_rows=P + 3), dict(src_row=P + 2)):
        assert call(p, params(**kw)) == ekv.ERR_INVALID_ARG, kw
    for kw in (dict(q=None), dict(out=None), dict(out=P), dict(q=P + 8), dict(out=P + 2), dict(ws=P + 4), dict(stride=511), dict(stride=516),
               dict(stride=-8)):
        assert call(p, params(), **kw) == ekv.ERR_INVALID_ARG, kw
    assert L.ekv_window_attention(None, C.byref(params()), P, 0, 2 * P, None, 0, None) == ekv.ERR_INVALID_ARG
    assert L.ekv_window_attention(p.h, None, P, 0, 2 * P, None, 0, None) == ekv.ERR_INVALID_ARG


@pytest.mark.parametrize("dim", [16, 32, 48, 80, 96, 112, 192, 224])
def test_other_head_dims(dim):
    assert call(pool(head_dim=dim), params(), stride=8 * dim) == ekv.ERR_UNSUPPORTED


def test_calls_without_rows_are_done():
    p = pool()
    assert call(p, params(n_batch=0)) == ekv.OK
    assert call(p, params(max_rows=0)) == ekv.OK


def test_rows_beyond_32_bits():
    """Rows of a KV head are counted in 32 bits."""
    p = pool()
    for kw in (dict(max_rows=2 ** 31 - 1), dict(max_rows=2 ** 30, q_heads=4), dict(max_rows=2 ** 20, q_heads=2 * 4096), dict(q_heads=2 * 8192)):
        assert L.ekv_window_attention(p.h, C.byref(params(**kw)), P, 0, 2 * P, None, 0, None) == ekv.ERR_UNSUPPORTED, kw
        assert L.ekv_window_attention_workspace_size(p.h, C.byref(params(**kw))) == 0, kw


def test_workspace_size():
    p = pool()

    def size(**kw):
        return L.ekv_window_attention_workspace_size(p.h, C.byref(params(**kw)))

    assert size() > 0 and size(max_rows=300) > 0
    for kw in (dict(n_batch=0), dict(n_batch=-1), dict(max_rows=0), dict(max_rows=-5), dict(q_heads=0), dict(q_heads=7)):
        assert size(**kw) == 0, kw
    assert L.ekv_window_attention_workspace_size(None, C.byref(params())) == 0
    assert L.ekv_window_attention_workspace_size(p.h, None) == 0


def test_binding_refuses_other_tensors():
    p = pool()
    i = torch.zeros(3, dtype=torch.int32)
    arg = dict(layer=0, seq_ids=i, dst_pos=i, n_rows=i, src_row=i, max_rows=5, q_heads=8, scale=0.125)
    prm = p.window_params(**arg)
    for name in ("seq_ids", "dst_pos", "n_rows", "src_row"):
        with pytest.raises(ValueError, match=name):
            p.window_params(**dict(arg, **{name: torch.zeros(3)}))
        if name != "seq_ids":
            with pytest.raises(ValueError, match=name):
                p.window_params(**dict(arg, **{name: torch.zeros(2, dtype=torch.int32)}))
    q = torch.zeros(9, 8, 64, dtype=torch.bfloat16)
    for bad_q, out in ((q, q[:8]), (q, q.float()), (q.float(), q.float()), (q.half(), q.half()), (q[:, :4], q[:, :4].contiguous()),
                       (q, torch.zeros(8, 9, 64, dtype=torch.bfloat16).transpose(0, 1))):
        with pytest.raises(ValueError):
            p.window_attention(prm, bad_q, out)
    with pytest.raises(ValueError):
        p.window_attention(prm, q, torch.empty_like(q), workspace=torch.zeros(64, 64, dtype=torch.uint8)[:, :8])
