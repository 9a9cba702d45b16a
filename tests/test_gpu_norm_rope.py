"""The rotary append with head norms on the GPU against 64-bit forms (decode_cases.py).

Tolerances. A result is rounded to bf16 once: half a step, 2^-8 of it at most. Before that: the mean of squares, its root and three
products in f32, 2^-20 of the value together; sine and cosine are off by 2^-21 of the pair's size. Pages of 8 bits hold what
ekv_append makes of the same bf16 rows."""
import pytest
import torch

import decode_cases as dc
import ekv

pytestmark = pytest.mark.gpu


def rand(seed, *shape, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).bfloat16().cuda()


def normed(x, weight, offset, eps):
    x = x.double()
    w = 1.0 if weight is None else weight.double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (w + offset)


def expect(x, weight, positions, rope, *, n, interleaved, offset, eps, after):
    """The value in 64 bits, and what it may be off by."""
    freq, mag = rope.frequencies()
    if after:
        y, size = dc.rope(x, positions, freq, n, interleaved, mag)
        f = normed(y, weight, offset, eps)
        size = size * ((f / y).abs().nan_to_num(0, 0, 0))
    else:
        f, size = dc.rope(normed(x, weight, offset, eps), positions, freq, n, interleaved, mag)
    return f, f.abs() * (2 ** -8 + 2 ** -20) + size * 2 ** -19 + 1e-37


def setup(store, dim, rows, hk, block=16, layers=1):
    c = dc.Cache([n + 2 for n in rows], hk, dim, store=store, block=block, layers=layers, seed=5)
    n_rows = dc.ints(rows)
    src = (n_rows.cumsum(0) - n_rows).int()
    return c, n_rows, src


@pytest.mark.parametrize("store,dim,rotary", [("bf16", 16, 16), ("bf16", 48, 48), ("bf16", 64, 64), ("bf16", 80, 34), ("bf16", 128, 128), ("bf16", 128, 64),
                                              ("bf16", 256, 66), ("bf16", 256, 256), ("q8_0", 32, 32), ("q8_0", 96, 48), ("q8_0", 128, 128),
                                              ("q8_0", 128, 6), ("q8_0", 224, 96), ("q8_0", 256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("after", [False, True])
def test_norm_rope_append(store, dim, rotary, interleaved, after):
    """Ragged requests, slices of one projection, odd head counts, positions far out."""
    rows, hq, hk = [7, 0, 33, 1], 5, 3
    c, n_rows, src = setup(store, dim, rows, hk)
    total = sum(rows)
    qkv = rand(dim, total + 1, (hq + 2 * hk) * dim, scale=3.0)[:total]
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([hq * dim, hk * dim, hk * dim], 1))
    offset = 1.0 if after else 0.0
    kind = torch.float32 if interleaved else torch.bfloat16
    qw, kw = (rand(i, dim).to(kind) for i in (1, 2))
    positions = (torch.arange(total) * 977 % 100003).int().cuda()
    rope = ekv.Rope(rotary_dims=rotary, interleaved=interleaved, attn_factor=1.25)
    norm = ekv.HeadNorm(q_weight=qw, k_weight=kw, eps=1e-5, weight_offset=offset, after_rotation=after)
    out = torch.full((total + 1, hq, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    before = [c.raw(b) for b in range(4)]
    c.pool.norm_rope_append(rope, norm, 0, c.seq_ids, dc.ints([2, 2, 1, 0]), n_rows, src, max(rows), positions, q=q, q_out=out[:total], k=k, v=v)
    assert c.pool.status() == 0
    kw_ = dict(n=rotary, interleaved=interleaved, offset=offset, eps=1e-5, after=after)
    want, tol = expect(q, qw, positions, rope, **kw_)
    assert ((out[:total].double() - want).abs() <= tol).all()
    assert (out[total] == 7.0).all()  # the row behind the last
    want, tol = expect(k, kw, positions, rope, **kw_)
    if store == "bf16":
        for b, at in enumerate([2, 2, 1, 0]):
            got_k, got_v = c.rows(b)
            s, e = int(src[b]), int(src[b]) + rows[b]
            assert ((got_k[at:at + rows[b]].double() - want[s:e]).abs() <= tol[s:e]).all()
            assert torch.equal(got_v[at:at + rows[b]].bfloat16(), v[s:e])
            now = c.raw(b)
            for x, y in zip(now, before[b]):  # rows before and behind
                w = hk * dim * 2
                assert torch.equal(x[:at * w], y[:at * w]) and torch.equal(x[(at + rows[b]) * w:], y[(at + rows[b]) * w:])
    else:
        # a bf16 pool holds the rows that are quantised: ekv_append of those gives the same bytes
        bf, _, _ = setup("bf16", dim, rows, hk)
        bf.pool.norm_rope_append(rope, norm, 0, bf.seq_ids, dc.ints([2, 2, 1, 0]), n_rows, src, max(rows), positions, k=k, v=v)
        ref, _, _ = setup("q8_0", dim, rows, hk)
        for b, at in enumerate([2, 2, 1, 0]):
            kk, vv = (x.bfloat16()[at:at + rows[b]].contiguous() for x in bf.rows(b))
            if rows[b]:
                ref.pool.append(0, ref.seq_ids[b:b + 1], dc.ints([at]), dc.ints([rows[b]]), dc.ints([0]), rows[b], kk, vv)
            for x, y in zip(c.raw(b), ref.raw(b)):
                assert torch.equal(x, y), b


@pytest.mark.parametrize("rows", [[1], [3, 1], [600, 100], [50] * 64])
@pytest.mark.parametrize("dim,hq,hk", [(256, 8, 1), (128, 32, 8), (64, 6, 2)])
def test_few_and_many_rows(rows, dim, hq, hk):
    """Rows shared by eight warps down to one; in place; q alone and k alone give the same as both."""
    c, n_rows, src = setup("bf16", dim, rows, hk)
    total = sum(rows)
    q, k, v = rand(1, total, hq, dim), rand(2, total, hk, dim), rand(3, total, hk, dim)
    qw, kw = rand(4, dim), rand(5, dim)
    positions = (torch.arange(total) % 5000).int().cuda()
    rope = ekv.Rope(rotary_dims=dim)
    norm = ekv.HeadNorm(q_weight=qw, k_weight=kw)
    zero = dc.ints([0] * len(rows))
    out = torch.empty_like(q)
    args = (rope, norm, 0, c.seq_ids, zero, n_rows, src, max(rows), positions)
    c.pool.norm_rope_append(*args, q=q, q_out=out, k=k, v=v)
    want, tol = expect(q, qw, positions, rope, n=dim, interleaved=False, offset=0.0, eps=1e-6, after=False)
    assert ((out.double() - want).abs() <= tol).all()
    pages = [c.raw(b) for b in range(len(rows))]
    c2, _, _ = setup("bf16", dim, rows, hk)
    both = torch.empty_like(q)
    c2.pool.norm_rope_append(*args, q=q, q_out=both)
    c2.pool.norm_rope_append(*args, k=k, v=v)
    assert torch.equal(both, out)
    q2 = q.clone()
    c2.pool.norm_rope_append(*args, q=q2, q_out=q2)
    assert torch.equal(q2, out)
    for b in range(len(rows)):
        assert all(torch.equal(x, y) for x, y in zip(pages[b], c2.raw(b)))
    assert c.pool.status() == 0 and c2.pool.status() == 0


def test_no_weights_zero_rows_and_scaled_contexts():
    c, n_rows, src = setup("bf16", 64, [3], 1)
    q = rand(1, 3, 2, 64)
    q[1] = 0
    positions = dc.ints([0, 123456, 9])
    rope = ekv.Rope(rotary_dims=64, freq_scale=0.25, ext_factor=1.0, n_ctx_orig=4096)
    norm = ekv.HeadNorm(eps=1e-6, weight_offset=0.5)
    out = torch.empty_like(q)
    c.pool.norm_rope_append(rope, norm, 0, c.seq_ids, dc.ints([0]), n_rows, src, 3, positions, q=q, q_out=out)
    want, tol = expect(q, None, positions, rope, n=64, interleaved=False, offset=0.5, eps=1e-6, after=False)
    assert ((out.double() - want).abs() <= tol).all() and (out[1] == 0).all()


def test_bad_rows_are_reported_and_others_done():
    c, n_rows, src = setup("bf16", 64, [4, 4, 4], 2)
    q, k, v = rand(1, 12, 4, 64), rand(2, 12, 2, 64), rand(3, 12, 2, 64)
    rope, norm = ekv.Rope(rotary_dims=64), ekv.HeadNorm()
    before = [c.raw(b) for b in range(3)]
    for ids, dst, code in (([c.seqs[0], 99, c.seqs[2]], [0, 0, 0], ekv.DEV_ERR_BAD_SEQ), ([c.seqs[0], c.seqs[1], -1], [0, 3, 0], None)):
        out = torch.zeros_like(q)
        c.pool.norm_rope_append(rope, norm, 0, dc.ints(ids), dc.ints(dst), n_rows, src, 4, dc.ints(range(12)), q=q, q_out=out, k=k, v=v)
        got = c.pool.status()
        assert got == code if code else got in (ekv.DEV_ERR_BAD_SEQ, ekv.DEV_ERR_BAD_POS)
        want, tol = expect(q, None, dc.ints(range(12)), rope, n=64, interleaved=False, offset=0.0, eps=1e-6, after=False)
        assert ((out.double() - want).abs() <= tol).all()
    # request 1's first three rows of the second call were inside its length (6 tokens), the fourth was not
    w = 2 * 64 * 2
    now = c.raw(1)
    assert torch.equal(now[0][:3 * w], before[1][0][:3 * w]) and not torch.equal(now[0][3 * w:], before[1][0][3 * w:])


def test_replayed_on_another_stream():
    c, n_rows, src = setup("q8_0", 128, [20, 5], 2)
    q, k, v = rand(1, 25, 8, 128), rand(2, 25, 2, 128), rand(3, 25, 2, 128)
    rope, norm = ekv.Rope(rotary_dims=128), ekv.HeadNorm(q_weight=rand(4, 128), k_weight=rand(5, 128))
    args = (rope, norm, 0, c.seq_ids, dc.ints([0, 1]), n_rows, src, 20, dc.ints(range(25)))
    out = torch.empty_like(q)
    c.pool.norm_rope_append(*args, q=q, q_out=out, k=k, v=v)
    pages = [c.raw(b) for b in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        c.pool.norm_rope_append(*args, q=q, q_out=out, k=k, v=v)
    want = out.clone()
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    for b in range(2):
        assert all(torch.equal(x, y) for x, y in zip(pages[b], c.raw(b)))


def test_weights_of_another_shape_are_refused():
    c, n_rows, src = setup("bf16", 64, [1], 1)
    with pytest.raises(ValueError):
        ekv.HeadNorm(q_weight=rand(1, 64), k_weight=rand(2, 32))
    with pytest.raises(ValueError):
        ekv.HeadNorm(q_weight=rand(1, 64).half())
    q = rand(1, 1, 2, 64)
    with pytest.raises(ValueError):
        c.pool.norm_rope_append(ekv.Rope(rotary_dims=64), ekv.HeadNorm(q_weight=rand(1, 32)), 0, c.seq_ids, dc.ints([0]), n_rows, src, 1,
                                dc.ints([0]), q=q, q_out=torch.empty_like(q))
