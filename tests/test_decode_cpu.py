"""Argument checks of the token-by-token decoding entry points and the rotary frequencies; no kernel is launched (the pool
is host-only, so a call that passes the checks ends with EKV_ERR_UNSUPPORTED)."""
import ctypes as C
import math

import numpy as np
import pytest

import decode_cases as dc
import ekv

P = 0x10000  # a pointer that is never followed
L = ekv.lib


def pool(**kw):
    cfg = dict(device=-1, dtype=ekv.DTYPE_BF16, block_tokens=16, n_blocks=40, kv_heads=2, head_dim=64, n_layers=2, max_seqs=6,
               max_blocks_per_seq=12)
    cfg.update(kw)
    return ekv.Pool(**cfg)


def tree_params(**kw):
    p = ekv.TreeParams(0, 3, 4, 8, 0.125, 0.0, ekv.DTYPE_BF16, 0, P, None, None, P)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def tree(p, prm, q=P, k=P, v=P, out=P, lse=P, ws=P):
    return L.ekv_tree_attention(p.h, C.byref(prm), q, k, v, out, lse, ws, 1 << 20, None)


def test_tree_attention_refusals():
    p = pool()
    assert tree(p, tree_params()) == ekv.ERR_UNSUPPORTED  # no device
    for kw in (dict(layer=2), dict(layer=-1), dict(n_batch=0), dict(n_draft=0), dict(q_heads=0), dict(q_heads=7), dict(scale=0.0),
               dict(scale=math.nan), dict(scale=math.inf), dict(softcap=-1.0), dict(softcap=math.nan), dict(seq_ids=None),
               dict(ancestors=P + 4)):
        assert tree(p, tree_params(**kw)) == ekv.ERR_INVALID_ARG, kw
    assert tree(p, tree_params(n_draft=65)) == ekv.ERR_RANGE
    assert tree(p, tree_params(out_dtype=ekv.DTYPE_F16)) == ekv.ERR_UNSUPPORTED
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=P + 8), dict(k=P + 2), dict(v=P + 2), dict(out=P + 8),
               dict(ws=P + 8), dict(lse=P + 2)):
        assert tree(p, tree_params(), **kw) == ekv.ERR_INVALID_ARG, kw
    assert tree(pool(head_dim=80), tree_params()) == ekv.ERR_UNSUPPORTED
    assert L.ekv_tree_attention(None, C.byref(tree_params()), P, P, P, P, None, None, 0, None) == ekv.ERR_INVALID_ARG
    assert L.ekv_tree_attention(p.h, None, P, P, P, P, None, None, 0, None) == ekv.ERR_INVALID_ARG


def test_tree_workspace_size():
    p = pool()
    assert L.ekv_tree_attention_workspace_size(p.h, C.byref(tree_params())) > 0
    for kw in (dict(n_draft=65), dict(n_draft=0), dict(q_heads=7), dict(n_batch=0)):
        assert L.ekv_tree_attention_workspace_size(p.h, C.byref(tree_params(**kw))) == 0
    assert L.ekv_tree_attention_workspace_size(None, C.byref(tree_params())) == 0


def test_key_weights_refusals():
    p = pool()

    def call(prm=None, q=P, lse=P, w=P, stride=100, decay=1.0):
        return L.ekv_key_weights(p.h, C.byref(prm or tree_params()), q, lse, w, stride, decay, None)

    assert call() == ekv.ERR_UNSUPPORTED
    for kw in (dict(q=None), dict(lse=None), dict(w=None), dict(stride=-1), dict(decay=math.nan), dict(w=P + 2), dict(lse=P + 1),
               dict(prm=tree_params(layer=5))):
        assert call(**kw) == ekv.ERR_INVALID_ARG, kw
    assert call(prm=tree_params(n_draft=65)) == ekv.ERR_RANGE


def test_evict_refusals():
    p = pool()

    def call(**kw):
        e = ekv.EvictParams(0, 2, 3, 32, 4, 8, P, None, P, None, 100, P, None, None, 0)
        for k, v in kw.items():
            setattr(e, k, v)
        return L.ekv_evict_by_weight(p.h, C.byref(e), None)

    assert call() == ekv.ERR_UNSUPPORTED
    for kw in (dict(layer0=-1), dict(layer0=1), dict(n_layers=0), dict(n_layers=3), dict(n_batch=0), dict(keep=0), dict(first=-1),
               dict(recent=-1), dict(first=16, recent=17), dict(first=2 ** 31 - 1, recent=2 ** 31 - 1), dict(weight_stride=-1),
               dict(seq_ids=None), dict(weights=None), dict(kept=None), dict(weights_out=P, out_stride=32),
               dict(positions=P, positions_out=P, out_stride=64), dict(weights_out=P + 4096, out_stride=31), dict(kept=P + 2)):
        assert call(**kw) == ekv.ERR_INVALID_ARG, kw
    assert call(weights_out=P, out_stride=100) == ekv.ERR_UNSUPPORTED
    big = pool(n_blocks=3000, block_tokens=256, max_blocks_per_seq=3000)
    s = big.seq_create()
    big.seq_resize(s, ekv.MAX_EVICT_TOKENS + 1)
    e = ekv.EvictParams(0, 1, 1, 32, 4, 8, P, None, P, None, 1 << 20, P, None, None, 0)
    assert L.ekv_evict_by_weight(big.h, C.byref(e), None) == ekv.ERR_RANGE


def test_rope_append_refusals():
    p, rope = pool(), ekv.Rope(device=-1, rotary_dims=64)

    def call(pl=None, r=None, layer=0, n=3, seq=P, dst=P, rows=P, src=P, most=5, pos=P, hq=4, q=P, qs=0, qo=P, k=P, v=P, kvs=0):
        return L.ekv_rope_append((pl or p).h, r or rope.h, layer, n, seq, dst, rows, src, most, pos, hq, q, qs, qo, k, v, kvs, None)

    assert call() == ekv.ERR_UNSUPPORTED
    assert call(n=0) == ekv.OK and call(most=0) == ekv.OK
    for kw in (dict(layer=2), dict(n=-1), dict(n=65536), dict(most=-1), dict(seq=None), dict(dst=None), dict(rows=None), dict(src=None),
               dict(pos=None), dict(hq=0), dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(q=None, qo=None, k=None, v=None),
               dict(qs=255), dict(qs=260), dict(kvs=127), dict(kvs=132), dict(q=P + 8, qo=P), dict(k=P + 2), dict(qs=512, qo=P)):
        assert call(**kw) == ekv.ERR_INVALID_ARG, kw
    assert call(qs=512, qo=P + 4096) == ekv.ERR_UNSUPPORTED
    assert call(pl=pool(head_dim=48)) == ekv.ERR_INVALID_ARG  # more rotated columns than a head has


@pytest.mark.parametrize("kw", [dict(rotary_dims=0), dict(rotary_dims=7), dict(rotary_dims=64, freq_base=1.0), dict(rotary_dims=64, freq_scale=0.0),
                                dict(rotary_dims=64, freq_scale=math.nan), dict(rotary_dims=64, ext_factor=1.0), dict(rotary_dims=64, ext_factor=-1.0),
                                dict(rotary_dims=64, ext_factor=1.0, n_ctx_orig=4096, beta_slow=0.0), dict(rotary_dims=64, attn_factor=math.inf),
                                dict(rotary_dims=4, freq_factors=[1.0, 0.0])])
def test_rope_create_refusals(kw):
    with pytest.raises(ekv.EkvError) as e:
        ekv.Rope(device=-1, **kw)
    assert e.value.code == ekv.ERR_INVALID_ARG
    with pytest.raises(ekv.EkvError) as e:
        ekv.Rope(device=-1, rotary_dims=258)
    assert e.value.code == ekv.ERR_UNSUPPORTED


@pytest.mark.parametrize("n", [2, 34, 64, 256])
@pytest.mark.parametrize("kw", [dict(), dict(freq_scale=0.25), dict(freq_base=1e6, freq_scale=0.125, ext_factor=1.0, n_ctx_orig=4096),
                                dict(freq_scale=0.5, ext_factor=0.25, n_ctx_orig=100, beta_fast=8.0, beta_slow=2.0)])
def test_rope_frequencies(n, kw):
    f, m = ekv.Rope(device=-1, rotary_dims=n, **kw).frequencies()
    want = dc.rope_table(n, kw.get("freq_base", 10000.0), kw.get("freq_scale", 1.0), kw.get("ext_factor", 0.0), kw.get("beta_fast", 32.0),
                         kw.get("beta_slow", 1.0), kw.get("n_ctx_orig", 0))
    np.testing.assert_allclose(f, want, rtol=1e-13)
    assert abs(m - (1 + 0.1 * math.log(1 / kw["freq_scale"]) if kw.get("ext_factor") else 1.0)) < 1e-6


def test_python_checks_of_rope_rows():
    torch = pytest.importorskip("torch")
    p, rope = pool(), ekv.Rope(device=-1, rotary_dims=64)
    x = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    n = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        p.rope_append(rope, 0, n, n, n, n, 3, n, q=x.transpose(0, 1), q_out=x)
    with pytest.raises(ValueError):
        p.rope_append(rope, 0, n, n, n, n, 3, n, q=x, q_out=x[:2])
    with pytest.raises(ValueError):
        p.rope_append(rope, 0, n, n, n, n, 3, n, k=x, v=x)  # 4 KV heads, the pool has 2


class NoStream:
    cuda_stream = 0


def test_python_checks_of_tree_layouts():
    """tree_attention and key_weights read and write adjacent rows: slices of a projection, short buffers and other types are
    refused; what passes reaches the library (which has no device here)."""
    torch = pytest.importorskip("torch")
    p = pool()
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    ids = torch.zeros(3, dtype=torch.int32)
    prm = p.tree_params(layer=0, seq_ids=ids, n_draft=2, q_heads=4, scale=0.125)
    proj = bf(6, 8, 64)  # q, k and v of one projection: 4 + 2 + 2 heads
    q, k, v = proj.split([4, 2, 2], 1)
    good = dict(q=q.contiguous(), k=k.contiguous(), v=v.contiguous(), out=bf(3, 2, 4, 64), lse=torch.zeros(3, 2, 4))

    def tree(ws=None, params=prm, **kw):
        a = {**good, **kw}
        p.tree_attention(params, a["q"], a["k"], a["v"], a["out"], a["lse"], ws, stream=NoStream)

    def weights(w=None, **kw):
        a = {**good, **kw}
        p.key_weights(prm, a["q"], a["lse"], torch.zeros(3, 2, 100) if w is None else w, stream=NoStream)

    for call in (tree, weights, lambda: tree(lse=None), lambda: tree(ws=torch.zeros(64, dtype=torch.uint8)), lambda: tree(q=bf(5, 2, 4, 64))):
        with pytest.raises(ekv.EkvError) as e:
            call()
        assert e.value.code == ekv.ERR_UNSUPPORTED
    for kw in (dict(q=q), dict(k=k), dict(v=v), dict(out=bf(3, 2, 64, 4).transpose(2, 3)), dict(lse=torch.zeros(3, 4, 2).transpose(1, 2)),
               dict(q=bf(5, 4, 64)), dict(k=bf(5, 2, 64)), dict(v=bf(5, 2, 64)), dict(out=bf(3, 2, 3, 64)), dict(lse=torch.zeros(3, 2, 3)),
               dict(q=torch.zeros(3, 2, 4, 64)), dict(k=torch.zeros(6, 2, 64)), dict(v=good["v"].half()), dict(out=torch.zeros(3, 2, 4, 64)),
               dict(lse=bf(3, 2, 4)), dict(ws=torch.zeros(64, 2, dtype=torch.uint8).T)):
        with pytest.raises(ValueError):
            tree(**kw)
    f32 = p.tree_params(layer=0, seq_ids=ids, n_draft=2, q_heads=4, scale=0.125, out_dtype=ekv.DTYPE_F32)
    with pytest.raises(ValueError):
        tree(params=f32)
    with pytest.raises(ekv.EkvError):
        tree(params=f32, out=torch.zeros(3, 2, 4, 64))
    for kw in (dict(q=q), dict(q=bf(5, 4, 64)), dict(lse=torch.zeros(3, 2, 3)), dict(w=torch.zeros(3, 100, 2).transpose(1, 2)),
               dict(w=torch.zeros(2, 2, 100)), dict(w=bf(3, 2, 100)), dict(lse=torch.zeros(3, 4, 2).transpose(1, 2))):
        with pytest.raises(ValueError):
            weights(**kw)


def test_python_checks_of_tree_params():
    torch = pytest.importorskip("torch")
    p = pool()
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    good = dict(seq_ids=i32(3), prefix_len=i32(3), n_nodes=i32(4), ancestors=torch.zeros(3, 2, dtype=torch.int64))
    p.tree_params(layer=0, n_draft=2, q_heads=4, scale=1.0, **good)
    p.tree_params(layer=0, n_draft=2, q_heads=4, scale=1.0, **{**good, "seq_ids": ekv.DevArray(P, 3)})
    for kw in (dict(seq_ids=i32(3, 2)[:, 0]), dict(prefix_len=i32(2)), dict(prefix_len=i32(6)[::2]), dict(n_nodes=i32(2)),
               dict(seq_ids=torch.zeros(3, dtype=torch.int64)), dict(n_nodes=torch.zeros(3, dtype=torch.int64)),
               dict(ancestors=torch.zeros(3, 4, dtype=torch.int64)[:, :2]), dict(ancestors=i32(3, 2)),
               dict(ancestors=torch.zeros(3, 1, dtype=torch.int64))):
        with pytest.raises(ValueError):
            p.tree_params(layer=0, n_draft=2, q_heads=4, scale=1.0, **{**good, **kw})


def test_python_checks_of_evict_buffers():
    """What the eviction reads and writes has room for all layers, requests and KV heads, in the layout that it is written in."""
    torch = pytest.importorskip("torch")
    p = pool()  # 2 layers, 2 KV heads
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    good = dict(seq_ids=i32(3), weights=torch.zeros(2, 3, 2, 100), kept=i32(2, 3, 2, 32), weights_out=torch.zeros(2, 3, 2, 40),
                positions=i32(2, 3, 2, 100), positions_out=i32(2, 3, 2, 40), seen=i32(3))

    def call(**kw):
        a = {**good, **kw}
        p.evict_by_weight(0, 2, a.pop("seq_ids"), a.pop("weights"), keep=32, first=4, recent=8, stream=NoStream, **a)

    for kw in (dict(), dict(weights_out=None, positions_out=None), dict(positions=None), dict(seen=None), dict(kept=i32(384)),
               dict(seq_ids=ekv.DevArray(P, 3)), dict(seq_ids=ekv.DevArray(P, 3), seen=ekv.DevArray(P, 3)),
               dict(weights_out=good["weights"], positions_out=good["positions"])):
        with pytest.raises(ekv.EkvError) as e:
            call(**kw)
        assert e.value.code == ekv.ERR_UNSUPPORTED, kw
    for kw in (dict(kept=i32(2, 3, 2, 31)), dict(kept=i32(2, 3, 2, 40)), dict(kept=i32(1, 3, 2, 32)), dict(kept=torch.zeros(2, 3, 2, 32)),
               dict(weights=torch.zeros(1, 3, 2, 100), positions=i32(1, 3, 2, 100)), dict(weights=i32(2, 3, 2, 100)),
               dict(positions=torch.zeros(2, 3, 2, 100)), dict(positions=i32(2, 3, 2, 99)), dict(weights_out=torch.zeros(2, 3, 1, 40)),
               dict(weights_out=i32(2, 3, 2, 40)), dict(positions_out=i32(2, 2, 2, 40)), dict(positions_out=i32(2, 3, 2, 41)),
               dict(positions_out=torch.zeros(2, 3, 2, 40)), dict(seen=i32(2)), dict(seen=torch.zeros(3, dtype=torch.int64)),
               dict(seq_ids=i32(3, 2)[:, 0]), dict(seq_ids=torch.zeros(3, dtype=torch.int64)), dict(seen=ekv.DevArray(P, 2)),
               dict(weights=torch.zeros(2, 3, 100, 2).transpose(2, 3))):
        with pytest.raises(ValueError):
            call(**kw)


def test_evict_range_is_of_the_calls_sequences():
    """A sequence beyond the limit that the call does not need does not refuse it."""
    p = pool(n_blocks=3000, block_tokens=256, max_blocks_per_seq=3000)
    seqs = [p.seq_create() for _ in range(4)]
    p.seq_resize(seqs[1], ekv.MAX_EVICT_TOKENS + 1)

    def call(n):
        e = ekv.EvictParams(0, 1, n, 32, 4, 8, P, None, P, None, 1 << 20, P, None, None, 0)
        return L.ekv_evict_by_weight(p.h, C.byref(e), None)

    assert call(3) == ekv.ERR_UNSUPPORTED
    assert call(4) == ekv.ERR_RANGE
    p.seq_resize(seqs[1], ekv.MAX_EVICT_TOKENS)
    assert call(4) == ekv.ERR_UNSUPPORTED


def test_evict_keep_near_the_end_of_32_bits():
    """Slot counters run up to a block of threads past keep; nothing is launched where that is beyond 32 bits."""
    p = pool()
    for keep, code in ((2 ** 31 - 1, ekv.ERR_RANGE), (2 ** 31 - 1024, ekv.ERR_RANGE), (2 ** 30, ekv.ERR_UNSUPPORTED)):
        e = ekv.EvictParams(0, 2, 3, keep, 4, 8, P, None, P, None, 100, P, None, None, 0)
        assert L.ekv_evict_by_weight(p.h, C.byref(e), None) == code


def test_tree_scales_and_heads_whose_products_overflow():
    """A scale, a cap or their quotient that is infinite in f32 (a score of 0 would be NaN), and head counts beyond 32 bits."""
    p = pool()
    for kw in (dict(scale=3e38), dict(softcap=3e38), dict(softcap=1e-45), dict(scale=1e20, softcap=1e-20)):
        assert tree(p, tree_params(**kw)) == ekv.ERR_INVALID_ARG, kw
    for kw in (dict(scale=2e38), dict(softcap=1e-30), dict(softcap=2e38)):
        assert tree(p, tree_params(**kw)) == ekv.ERR_UNSUPPORTED, kw
    huge = tree_params(q_heads=2 ** 31 - 2, n_draft=64)
    assert tree(p, huge) == ekv.ERR_UNSUPPORTED
    assert L.ekv_tree_attention_workspace_size(p.h, C.byref(huge)) == 0
    assert L.ekv_tree_attention_workspace_size(p.h, C.byref(tree_params(q_heads=2 * 8191))) > 0


def test_tree_max_prefix_refusals():
    p = pool()
    assert tree(p, tree_params(max_prefix=-1)) == ekv.ERR_INVALID_ARG
    assert tree(p, tree_params(max_prefix=1)) == tree(p, tree_params(max_prefix=2 ** 31 - 1)) == ekv.ERR_UNSUPPORTED
