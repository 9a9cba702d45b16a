"""Token-by-token decoding operators on the GPU against plain 64-bit forms (decode_cases.py).

Tolerances. Rounding to the 8 significant bits of bf16 is off by at most 2^-8 of the value. Attention rounds each
probability so once, which puts an output off by at most 2^-8 of A = sum p |v|; a bf16 output adds 2^-8 of its own size,
at most A. A quarter on top is left for the f32 scores and
exponentials (head_dim * 2^-24 of sum |q k| <= 1e-3 here). lse and key weights see the f32 scores alone: an error of
head_dim * 2^-24 * max sum |q k| in a score, and 1e-5 for the exponential, the logarithm and the sums. A turned value is
rounded to bf16 once (2^-8 of it), and its sine and cosine are off by 2^-21 at most."""
import math

import numpy as np
import pytest
import torch

import decode_cases as dc
import ekv

pytestmark = pytest.mark.gpu


def run_tree(c, q, kd, vd, *, nodes=None, up=None, cap=0.0, dtype=torch.bfloat16, prefix_len=None, workspace=True, stream=None):
    B, T, hq, d = q.shape
    prm = c.pool.tree_params(layer=0, seq_ids=c.seq_ids, n_draft=T, q_heads=hq, scale=1 / math.sqrt(d), softcap=cap,
                             out_dtype=ekv.DTYPE_BF16 if dtype == torch.bfloat16 else ekv.DTYPE_F32,
                             prefix_len=None if prefix_len is None else dc.ints(prefix_len),
                             n_nodes=None if nodes is None else dc.ints(nodes), ancestors=up)
    out = torch.full((B, T, hq, d), 77.0, dtype=dtype, device="cuda")
    lse = torch.full((B, T, hq), 77.0, device="cuda")
    ws = torch.full((c.pool.tree_attention_workspace_size(prm),), 255, dtype=torch.uint8, device="cuda") if workspace else None
    if stream is not None:  # the buffers were filled on the current one
        stream.wait_stream(torch.cuda.current_stream())
    c.pool.tree_attention(prm, q, kd, vd, out, lse, ws, stream=stream)
    torch.cuda.synchronize()
    assert c.pool.status() == 0
    return out, lse, prm


def check_tree(c, q, kd, vd, out, lse, *, nodes=None, up=None, cap=0.0, prefix_len=None):
    B, T, hq, d = q.shape
    for b in range(B):
        n = c.lens[b] if prefix_len is None else prefix_len[b]
        k, v = c.rows(b, n=n)
        m = T if nodes is None else nodes[b]
        w = [(2 << t) - 1 for t in range(T)] if up is None else up[b]
        want, want_lse, size, most = dc.tree_attention(q[b], k, v, kd[b], vd[b], w, m, 1 / math.sqrt(d), cap)
        tol = (1.25 * 2 ** -7 if out.dtype == torch.bfloat16 else 1.25 * 2 ** -8) * size + 1e-30
        got = out[b].double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
        bad = ((got - want).abs() > tol) & fine & torch.isfinite(size)
        assert not bad.any(), (b, (got - want).abs().max().item(), bad.nonzero()[:3].tolist())
        empty = torch.isneginf(want_lse)
        assert torch.equal(torch.isneginf(lse[b]), empty)
        off = (lse[b].double() - want_lse).abs() - (d * 2 ** -24 * most + 1e-5 * (1 + want_lse.abs()))
        assert not (off[~empty] > 0).any(), off[~empty].max().item()


def rand(seed, *shape, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).bfloat16().cuda()


STORES = [("bf16", 48), ("bf16", 64), ("bf16", 128), ("bf16", 256), ("q8_0", 64), ("q8_0", 128), ("q8_0", 256)]


@pytest.mark.parametrize("store,dim", STORES)
@pytest.mark.parametrize("T,hq,hk", [(1, 4, 4), (1, 8, 1), (3, 6, 2), (5, 4, 1), (11, 12, 4), (17, 2, 1), (33, 4, 2), (64, 8, 1)])
def test_tree_attention(store, dim, T, hq, hk):
    lens = [333, 0, 64, 1, 127, 16]
    c = dc.Cache(lens, hk, dim, store=store, seed=dim + T)
    B = len(lens)
    q, kd, vd = rand(1, B, T, hq, dim, scale=1.5), rand(2, B, T, hk, dim), rand(3, B, T, hk, dim)
    nodes = [max(0, T - b) for b in range(B)]
    up = [dc.tree_words(T, b) for b in range(B)]
    for ws in (True, False):
        out, lse, _ = run_tree(c, q, kd, vd, nodes=nodes, up=dc.words(up), workspace=ws)
        check_tree(c, q, kd, vd, out, lse, nodes=nodes, up=up)


@pytest.mark.parametrize("block", [8, 16, 24, 40, 64, 128, 256])
@pytest.mark.parametrize("store", ["bf16", "q8_0"])
def test_tree_blocks_and_chain(store, block):
    """Pages that end inside tiles, a chain of drafts by default, f32 output."""
    c = dc.Cache([515, 200, 63], 2, 64, store=store, block=block, seed=block)
    q, kd, vd = rand(4, 3, 5, 4, 64), rand(5, 3, 5, 2, 64), rand(6, 3, 5, 2, 64)
    out, lse, _ = run_tree(c, q, kd, vd, dtype=torch.float32)
    check_tree(c, q, kd, vd, out, lse)


@pytest.mark.parametrize("store,dim", [("bf16", 128), ("q8_0", 128), ("bf16", 256)])
@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0])
def test_tree_long_ragged_capped(store, dim, cap):
    """Lengths that split over many CTAs beside short ones, capped scores, prefix_len below the length."""
    lens = [9001, 3, 0, 4097, 640]
    use = [9001, 2, 0, 4000, 1]
    c = dc.Cache(lens, 2, dim, store=store, block=32, seed=7)
    q, kd, vd = rand(8, 5, 6, 8, dim, scale=4.0), rand(9, 5, 6, 2, dim), rand(10, 5, 6, 2, dim)
    up = [dc.tree_words(6, 40 + b) for b in range(5)]
    out, lse, _ = run_tree(c, q, kd, vd, up=dc.words(up), cap=cap, prefix_len=use)
    check_tree(c, q, kd, vd, out, lse, up=up, cap=cap, prefix_len=use)


@pytest.mark.parametrize("store,dim", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("q8_0", 128)])
@pytest.mark.parametrize("T,hq,cap,dtype", [(64, 8, 20.0, torch.bfloat16), (19, 8, 0.0, torch.float32), (43, 3, 0.0, torch.bfloat16)])
def test_tree_wide_long_ragged(store, dim, T, hq, cap, dtype):
    """Many rows per KV head over caches of several tiles: rising maxima, odd row counts, parts of units, an empty cache."""
    lens = [3000, 0, 515, 129]
    c = dc.Cache(lens, 2, dim, store=store, block=24, seed=11)
    B = len(lens)
    q, kd, vd = rand(8, B, T, 2 * hq, dim, scale=5.0), rand(9, B, T, 2, dim), rand(10, B, T, 2, dim)
    nodes = [T, T - 1, 1, 0]
    up = [dc.tree_words(T, 60 + b) for b in range(B)]
    for ws in (True, False):
        out, lse, _ = run_tree(c, q, kd, vd, nodes=nodes, up=dc.words(up), cap=cap, dtype=dtype, workspace=ws)
        check_tree(c, q, kd, vd, out, lse, nodes=nodes, up=up, cap=cap)


def test_tree_rows_that_see_nothing():
    """Ancestor words of zero over an empty cache, no nodes at all: 0 and -inf."""
    c = dc.Cache([0, 40, 0], 1, 64, seed=1)
    q, kd, vd = rand(1, 3, 4, 2, 64), rand(2, 3, 4, 1, 64), rand(3, 3, 4, 1, 64)
    up = [[0, 2, 0, 8], [0, 0, 0, 0], [1, 2, 4, 8]]
    for ws in (True, False):
        out, lse, _ = run_tree(c, q, kd, vd, up=dc.words(up), nodes=[4, 4, 0], workspace=ws)
        check_tree(c, q, kd, vd, out, lse, up=up, nodes=[4, 4, 0])
        assert (out[0, 0] == 0).all() and torch.isneginf(lse[0, 0]).all()
        assert (out[2] == 0).all() and torch.isneginf(lse[2]).all()


@pytest.mark.parametrize("store,dim,T,hq", [("bf16", 64, 7, 2), ("q8_0", 128, 7, 2), ("bf16", 128, 20, 4), ("q8_0", 64, 40, 2), ("bf16", 256, 9, 8)])
def test_tree_hidden_values_do_not_leak(store, dim, T, hq):
    """Drafted keys and values of infinity and NaN reach the rows that see them and no others; unused drafts, rows past
    the cache's end and stale pages do not matter."""
    c = dc.Cache([70, 5], 1, dim, store=store, block=16, seed=3)
    q, kd, vd = rand(1, 2, T, hq, dim), rand(2, 2, T, 1, dim), rand(3, 2, T, 1, dim)
    nodes = [T - 2, T - 1]
    vd[:, 1, 0, 3] = float("inf")
    vd[:, 2, 0, dim - 1] = float("nan")
    vd[0, 4, 0, :9] = float("-inf")
    kd[:, 3, 0, 5] = float("nan")
    vd[:, T - 1], kd[:, T - 1] = float("nan"), float("inf")
    up = [[1 << t | (2 if t >= 5 else 0) | (1 if t % 2 else 0) for t in range(T)] for _ in range(2)]
    if store == "bf16":  # rows past the end of the last page: whatever an earlier request left there
        nan = torch.full((16, 1, dim), float("nan"), dtype=torch.bfloat16, device="cuda")
        for s, n in zip(c.seqs, c.lens):
            c.pool.seq_resize(s, -(-n // 16) * 16)
        c.pool.sync()
        tail = [-(-n // 16) * 16 - n for n in c.lens]
        c.pool.append(0, c.seq_ids, dc.ints(c.lens), dc.ints(tail), dc.ints([0, 0]), 16, nan, nan)
        for s, n in zip(c.seqs, c.lens):
            c.pool.seq_resize(s, n)
        c.pool.sync()
    out, lse, _ = run_tree(c, q, kd, vd, up=dc.words(up), nodes=nodes)
    for b in range(2):
        for t in range(nodes[b]):
            row = out[b, t].float()
            if t == 3:
                assert torch.isnan(row).all()
                continue
            sees = [j for j in range(nodes[b]) if up[b][t] >> j & 1]
            k, v = c.rows(b)
            kk = torch.cat([k, kd[b][sees].float()]).double()
            vv = torch.cat([v, vd[b][sees].float()]).double()
            s = torch.einsum("hd,kd->hk", q[b, t].double(), kk[:, 0]) / math.sqrt(dim)
            p = torch.softmax(s, -1)
            want = p @ vv[:, 0]
            same = torch.isnan(want) == torch.isnan(row.double())
            assert same.all()
            inf = torch.isinf(want)
            assert torch.equal(want[inf], row.double()[inf])
            fine = torch.isfinite(want)
            bound = 1.25 * 2 ** -7 * (p @ torch.nan_to_num(vv[:, 0], 0, 0, 0).abs())
            assert ((row.double() - want).abs()[fine] <= bound[fine]).all()


def test_tree_other_stream_and_repeats():
    """On a stream of its own, twice: the same bits."""
    c = dc.Cache([2000, 900], 2, 128, seed=5)
    q, kd, vd = rand(1, 2, 3, 8, 128), rand(2, 2, 3, 2, 128), rand(3, 2, 3, 2, 128)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    a = run_tree(c, q, kd, vd, stream=s)
    b = run_tree(c, q, kd, vd, stream=s)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    check_tree(c, q, kd, vd, *a[:2])


def test_tree_graph_capture():
    c = dc.Cache([700], 1, 64, seed=6)
    q, kd, vd = rand(1, 1, 2, 4, 64), rand(2, 1, 2, 1, 64), rand(3, 1, 2, 1, 64)
    out, lse, prm = run_tree(c, q, kd, vd)
    ws = torch.empty(c.pool.tree_attention_workspace_size(prm), dtype=torch.uint8, device="cuda")
    again = torch.zeros_like(out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.pool.tree_attention(prm, q, kd, vd, again, None, ws)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, out)


def test_tree_reports_bad_sequences():
    c = dc.Cache([64], 1, 64, seed=6)
    q, kd, vd = rand(1, 1, 1, 1, 64), rand(2, 1, 1, 1, 64), rand(3, 1, 1, 1, 64)
    prm = c.pool.tree_params(layer=0, seq_ids=dc.ints([9]), n_draft=1, q_heads=1, scale=1.0)
    out = torch.empty(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    c.pool.tree_attention(prm, q, kd, vd, out)
    torch.cuda.synchronize()
    assert c.pool.status() == ekv.DEV_ERR_BAD_SEQ
    prm = c.pool.tree_params(layer=0, seq_ids=c.seq_ids, n_draft=1, q_heads=1, scale=1.0, prefix_len=dc.ints([65]))
    c.pool.tree_attention(prm, q, kd, vd, out)
    torch.cuda.synchronize()
    assert c.pool.status() == ekv.DEV_ERR_BAD_POS


# ---------------------------------------------------------------------------------------------- key weights


@pytest.mark.parametrize("store,dim", STORES)
@pytest.mark.parametrize("T,hq,hk", [(1, 4, 4), (1, 8, 1), (13, 6, 2), (64, 8, 1)])
@pytest.mark.parametrize("decay,cap", [(0.0, 0.0), (1.0, 0.0), (0.5, 20.0)])
def test_key_weights(store, dim, T, hq, hk, decay, cap):
    lens = [333, 0, 64, 1, 1000]
    c = dc.Cache(lens, hk, dim, store=store, seed=dim + T)
    B = len(lens)
    q, kd, vd = rand(1, B, T, hq, dim, scale=1.5), rand(2, B, T, hk, dim), rand(3, B, T, hk, dim)
    nodes = [max(0, T - b) for b in range(B)]
    _, lse, prm = run_tree(c, q, kd, vd, nodes=nodes, cap=cap)
    w = torch.rand(B, hk, 1007, generator=torch.Generator().manual_seed(4)).cuda()
    if decay == 0.0:
        w[:] = float("nan")
    old = w.clone()
    c.pool.key_weights(prm, q, lse, w, decay)
    again = old.clone()
    c.pool.key_weights(prm, q, lse, again, decay)
    torch.cuda.synchronize()
    assert c.pool.status() == 0
    assert torch.equal(w.view(torch.int32), again.view(torch.int32))  # the same bits
    for b in range(B):
        n = lens[b]
        assert torch.equal(w[b, :, n:].view(torch.int32), old[b, :, n:].view(torch.int32))
        if n == 0:
            continue
        k, _ = c.rows(b)
        s, size = dc.tree_scores(q[b, :nodes[b]].double(), k.double(), 1 / math.sqrt(dim), cap)
        got = torch.exp(s - lse[b, :nodes[b]].double()[..., None]).unflatten(1, (hk, hq // hk)).sum((0, 2))
        want = got + (decay * old[b, :, :n].double() if decay else 0.0)
        tol = got * (dim * 2 ** -24 * (size.max().item() if size.numel() else 0) + 2e-5) + want * 1e-6 + 1e-30
        assert ((w[b, :, :n].double() - want).abs() <= tol).all()


def test_key_weights_rows_of_nothing_and_short_stride():
    c = dc.Cache([80], 1, 64, seed=2)
    q = rand(1, 1, 2, 2, 64)
    q[0, 1] = float("nan")
    lse = torch.tensor([[[1.0, -math.inf], [math.nan, math.nan]]], device="cuda")
    prm = c.pool.tree_params(layer=0, seq_ids=c.seq_ids, n_draft=2, q_heads=2, scale=0.125, n_nodes=dc.ints([1]))
    w = torch.zeros(1, 1, 80, device="cuda")
    c.pool.key_weights(prm, q, lse, w, 1.0)
    torch.cuda.synchronize()
    k, _ = c.rows(0)
    want = torch.exp(k[:, 0].double() @ q[0, 0, 0].double() * 0.125 - 1.0)
    assert ((w[0, 0].double() - want).abs() <= 1e-4 * want).all()
    assert c.pool.status() == 0
    short = torch.zeros(1, 1, 50, device="cuda")
    c.pool.key_weights(prm, q, lse, short, 1.0)
    torch.cuda.synchronize()
    assert c.pool.status() == ekv.DEV_ERR_BAD_POS
    assert torch.equal(short[0, 0], w[0, 0, :50])


# ---------------------------------------------------------------------------------------------- eviction


def check_evict(c, w, keep, first, recent, positions=None, seen=None, in_place=False):
    L, B, H, W = w.shape
    before = [[[x.clone() for x in c.raw(b, layer)] for b in range(B)] for layer in range(L)]
    kept = torch.full((L, B, H, keep), -7, dtype=torch.int32, device="cuda")
    w_in, p_in = w.clone(), None if positions is None else positions.clone()
    w_out = w if in_place else torch.full((L, B, H, keep + 3), 7.0, device="cuda")
    p_out = positions if in_place else torch.full((L, B, H, keep + 3), 7, dtype=torch.int32, device="cuda")
    c.pool.evict_by_weight(0, L, c.seq_ids, w, keep=keep, first=first, recent=recent, kept=kept, weights_out=w_out,
                           positions=positions, positions_out=p_out, seen=None if seen is None else dc.ints(seen))
    torch.cuda.synchronize()
    assert c.pool.status() == 0
    for layer in range(L):
        for b in range(B):
            n = c.lens[b]
            m = min(n, keep)
            after = c.raw(b, layer)
            for h in range(H):
                wl = w_in[layer, b, h, :n].tolist()
                pl = None if p_in is None else p_in[layer, b, h, :n].tolist()
                want = dc.evict(wl, n, keep, first, recent, pl, None if seen is None else seen[b])
                assert kept[layer, b, h].tolist() == want, (layer, b, h)
                at = torch.tensor(want[:m], dtype=torch.int64, device="cuda")
                assert torch.equal(w_out[layer, b, h, :m].view(torch.int32), w_in[layer, b, h][at].view(torch.int32))
                if p_out is not None:
                    assert torch.equal(p_out[layer, b, h, :m], (at.int() if p_in is None else p_in[layer, b, h][at]))
                    assert (p_out[layer, b, h, m:keep] == -1).all()
                assert (w_out[layer, b, h, m:keep] == 0).all()
                for x, y in zip(before[layer][b], after):
                    x, y = x.view(n, H, -1), y.view(n, H, -1)
                    assert torch.equal(y[:m, h], x[at, h])
                    if n > keep:
                        assert torch.equal(y[keep:, h], x[keep:, h])
    return kept


@pytest.mark.parametrize("store,dim,block", [("bf16", 48, 16), ("bf16", 64, 24), ("bf16", 128, 64), ("bf16", 256, 8), ("bf16", 32, 16),
                                             ("q8_0", 32, 16), ("q8_0", 64, 24), ("q8_0", 128, 64), ("q8_0", 256, 16)])
def test_evict(store, dim, block):
    lens = [300, 41, 40, 1, 129]
    c = dc.Cache(lens, 2, dim, store=store, block=block, layers=2, seed=dim)
    g = torch.Generator().manual_seed(dim)
    w = torch.exp(torch.randn(2, 5, 2, 307, generator=g)).cuda()
    w *= (torch.rand(w.shape, generator=g) > 0.3).cuda()  # ties at zero
    check_evict(c, w, 40, 4, 10)


@pytest.mark.parametrize("n,keep,first,recent", [(33, 32, 0, 0), (33, 32, 32, 0), (65, 1, 0, 1), (64, 63, 0, 63), (2100, 2048, 4, 100),
                                                 (5000, 7, 3, 4), (4100, 2049, 0, 0), (70000, 33000, 10, 1000)])
def test_evict_sizes(n, keep, first, recent):
    c = dc.Cache([n], 1, 32, block=32, seed=n)
    w = torch.rand(1, 1, 1, n, generator=torch.Generator().manual_seed(n)).cuda()
    w[0, 0, 0, ::3] = 0.25  # many ties, also where the choice ends
    check_evict(c, w, keep, first, recent)


def test_evict_weights_of_all_kinds():
    c = dc.Cache([200], 1, 64, seed=1)
    w = torch.randn(1, 1, 1, 200, generator=torch.Generator().manual_seed(2)).cuda()
    for i, x in enumerate([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42, -1e-42, math.nan]):
        w[0, 0, 0, 7 * i + 3] = x
    check_evict(c, w, 100, 0, 0)
    same = torch.ones(1, 1, 1, 200, device="cuda")
    check_evict(c, same, 100, 0, 50)
    none = torch.full((1, 1, 1, 200), math.nan, device="cuda")
    check_evict(c, none, 77, 3, 9)


def test_evict_twice_in_place_with_positions():
    """A second eviction goes by the positions that the first left in each slot; lengths shrink in between."""
    c = dc.Cache([150, 90], 2, 64, block=16, seed=9, width=12)
    g = torch.Generator().manual_seed(3)
    w = torch.rand(1, 2, 2, 160, generator=g).cuda()
    pos = torch.arange(160, dtype=torch.int32, device="cuda").repeat(1, 2, 2, 1).contiguous()
    check_evict(c, w, 100, 4, 30, positions=pos, seen=[150, 90], in_place=True)
    for b, s in enumerate(c.seqs):
        c.lens[b] = min(c.lens[b], 100)
        c.pool.seq_resize(s, c.lens[b])
        c.pool.seq_append_tokens(s, 20)
        c.lens[b] += 20
    c.pool.sync()
    k, v = rand(1, 20, 2, 64), rand(2, 20, 2, 64)
    c.pool.append(0, c.seq_ids, dc.ints([n - 20 for n in c.lens]), dc.ints([20, 20]), dc.ints([0, 0]), 20, k, v)
    for b, seen in enumerate([150, 90]):
        n = c.lens[b]
        pos[0, b, :, n - 20:n] = torch.arange(seen, seen + 20, dtype=torch.int32, device="cuda")
        w[0, b, :, n - 20:n] = 0.0
    check_evict(c, w, 100, 4, 30, positions=pos, seen=[170, 110], in_place=True)


def test_evict_reports_short_stride():
    c = dc.Cache([100], 1, 64, seed=1)
    w = torch.rand(1, 1, 1, 60, device="cuda")
    kept = torch.zeros(1, 1, 1, 50, dtype=torch.int32, device="cuda")
    c.pool.evict_by_weight(0, 1, c.seq_ids, w, keep=50, first=0, recent=0, kept=kept)
    torch.cuda.synchronize()
    assert c.pool.status() == ekv.DEV_ERR_BAD_POS
    assert (kept == -1).all()


# ---------------------------------------------------------------------------------------------- rotary append


def rope_case(store, dim, rotary, interleaved, lens, hq, hk, *, strided, positions=None, seed=0, **kw):
    """Rows to positions 3 .. of each request. Returns the cache, inputs and turned q."""
    c = dc.Cache([n + 3 for n in lens], hk, dim, store=store, seed=seed)
    rope = ekv.Rope(rotary_dims=rotary, interleaved=interleaved, **kw)
    total = sum(lens)
    pad = 24 if strided else 0
    qkv = rand(seed + 1, total, (hq + 2 * hk) * dim + pad)
    q = qkv[:, pad:pad + hq * dim].unflatten(1, (hq, dim))
    k = qkv[:, pad + hq * dim:pad + (hq + hk) * dim].unflatten(1, (hk, dim))
    v = qkv[:, pad + (hq + hk) * dim:].unflatten(1, (hk, dim))
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    pos = torch.arange(total, device="cuda", dtype=torch.int32) * 7 % 4001 if positions is None else dc.ints(positions)
    out = torch.zeros(total, hq, dim, dtype=torch.bfloat16, device="cuda")
    start = dc.ints(np.cumsum([0] + lens[:-1]))
    c.pool.rope_append(rope, 0, c.seq_ids, dc.ints([3] * len(lens)), dc.ints(lens), start, max(lens), pos, q=q, q_out=out, k=k, v=v)
    torch.cuda.synchronize()
    assert c.pool.status() == 0
    return c, rope, q, k, v, pos, out


def close_turned(got, want, size):
    tol = want.abs() * 2 ** -7.99 + size * 2 ** -20 + 1e-38
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), ((got.double() - want).abs() - tol).max().item()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("store,dim,rotary", [("bf16", 48, 48), ("bf16", 64, 18), ("bf16", 128, 128), ("bf16", 256, 64), ("bf16", 112, 34), ("bf16", 16, 2),
                                              ("q8_0", 64, 64), ("q8_0", 128, 34), ("q8_0", 256, 256), ("q8_0", 96, 48)])
@pytest.mark.parametrize("strided", [False, True])
def test_rope_append(store, dim, rotary, interleaved, strided):
    lens, hq, hk = [1, 37, 16, 3], 6, 2
    c, rope, q, k, v, pos, out = rope_case(store, dim, rotary, interleaved, lens, hq, hk, strided=strided, seed=dim + rotary)
    freq, mag = rope.frequencies()
    np.testing.assert_allclose(freq, dc.rope_table(rotary), rtol=1e-14)
    assert mag == 1.0
    close_turned(out, *dc.rope(q, pos, freq, rotary, interleaved))
    # the pages hold what ekv_append of the turned rows writes, bit for bit; rows 0 .. 2 are untouched
    turned = torch.zeros(k.shape, dtype=torch.bfloat16, device="cuda")
    zeros = dc.ints([0] * len(lens))
    start = dc.ints(np.cumsum([0] + lens[:-1]))
    c.pool.rope_append(rope, 0, None, None, dc.ints(lens), start, max(lens), pos, q=k, q_out=turned)
    close_turned(turned, *dc.rope(k, pos, freq, rotary, interleaved))
    other = dc.Cache([n + 3 for n in lens], hk, dim, store=store, seed=dim + rotary)
    other.pool.append(0, other.seq_ids, zeros + 3, dc.ints(lens), start, max(lens), turned, v.contiguous())
    torch.cuda.synchronize()
    for b in range(len(lens)):
        for x, y in zip(c.raw(b), other.raw(b)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("kw", [dict(freq_scale=0.25), dict(freq_scale=0.125, ext_factor=1.0, n_ctx_orig=4096),
                                dict(freq_scale=0.25, ext_factor=0.5, n_ctx_orig=2048, attn_factor=0.8, beta_fast=16.0, beta_slow=2.0),
                                dict(freq_base=500000.0, freq_factors=[1.0 + 0.25 * i for i in range(32)])])
def test_rope_long_contexts(kw):
    """Positions to beyond 2^24, scaled frequencies: the angle must not lose what 32 bits would."""
    pos = [0, 1, 4095, 100000, 1 << 20, (1 << 24) + 1, 2 ** 31 - 1, 77, -5]
    c, rope, q, k, v, p, out = rope_case("bf16", 64, 64, False, [9], 3, 1, strided=True, positions=pos, **kw)
    freq, mag = rope.frequencies()
    ff = kw.get("freq_factors")
    want = dc.rope_table(64, kw.get("freq_base", 10000.0), kw.get("freq_scale", 1.0), kw.get("ext_factor", 0.0), kw.get("beta_fast", 32.0),
                         kw.get("beta_slow", 1.0), kw.get("n_ctx_orig", 0), ff)
    np.testing.assert_allclose(freq, want, rtol=1e-13)
    m = kw.get("attn_factor", 1.0) * (1 + 0.1 * math.log(1 / kw["freq_scale"]) if kw.get("ext_factor") else 1.0)
    assert abs(mag - m) < 1e-6
    close_turned(out, *dc.rope(q, p, freq, 64, False, mag))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_in_place_and_append_only(interleaved):
    c, rope, q, k, v, pos, out = rope_case("bf16", 64, 32, interleaved, [20, 9], 4, 2, strided=False)
    q2 = q.clone()
    c.pool.rope_append(rope, 0, None, None, dc.ints([20, 9]), dc.ints([0, 20]), 20, pos, q=q2, q_out=q2)
    torch.cuda.synchronize()
    assert torch.equal(q2, out)
    other = dc.Cache([23, 12], 2, 64)
    other.pool.rope_append(rope, 0, other.seq_ids, dc.ints([3, 3]), dc.ints([20, 9]), dc.ints([0, 20]), 20, pos, k=k, v=v)
    torch.cuda.synchronize()
    for b in range(2):
        for x, y in zip(c.raw(b), other.raw(b)):
            assert torch.equal(x[3 * 256:], y[3 * 256:])


def test_rope_append_reports_bad_places():
    c = dc.Cache([10], 1, 64)
    rope = ekv.Rope(rotary_dims=64)
    k, v = rand(1, 4, 1, 64), rand(2, 4, 1, 64)
    before = [x.clone() for x in c.raw(0)]
    pos = dc.ints([0, 1, 2, 3])
    c.pool.rope_append(rope, 0, c.seq_ids, dc.ints([8]), dc.ints([4]), dc.ints([0]), 4, pos, k=k, v=v)
    torch.cuda.synchronize()
    assert c.pool.status() == ekv.DEV_ERR_BAD_POS
    for x, y in zip(before, c.raw(0)):
        assert torch.equal(x[:8 * 128], y[:8 * 128]) and not torch.equal(x, y)
    c.pool.rope_append(rope, 0, dc.ints([55]), dc.ints([0]), dc.ints([1]), dc.ints([0]), 1, pos, k=k, v=v)
    torch.cuda.synchronize()
    assert c.pool.status() == ekv.DEV_ERR_BAD_SEQ
