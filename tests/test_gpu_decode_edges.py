"""Decoding operators where inputs are not finite, and what rounding may not cost. Shapes, checks and tolerances not derived
here are those of test_gpu_decode.py."""
import math

import pytest
import torch

import decode_cases as dc
import ekv
from test_gpu_decode import STORES, check_evict, check_tree, close_turned, rand, run_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store,dim", STORES)
@pytest.mark.parametrize("T,hq", [(1, 4), (3, 5), (6, 4), (45, 4)])
@pytest.mark.parametrize("cap", [0.0, 9.0])
def test_tree_rows_without_a_number_stay_so(store, dim, T, hq, cap):
    """A row whose every score is NaN (its query is, or the one key that it sees) gives NaN, as the formula does, not the 0
    and -inf of a row that sees nothing; short and long caches, with the cache cut into parts and without."""
    lens = [0, 0, 40, 900, 5000]
    c = dc.Cache(lens, 1, dim, store=store, seed=dim)
    B = len(lens)
    q, kd, vd = rand(61, B, T, hq, dim), rand(62, B, T, 1, dim), rand(63, B, T, 1, dim)
    q[0, 0, 1, 3] = float("nan")
    kd[1, T - 1, 0, 5] = float("nan")
    q[2:, T - 1, hq - 1, 7] = float("nan")
    q[4, T // 2] = float("nan")
    up = [[1 << t for t in range(T)] for _ in range(B)]
    for ws in (True, False):
        for nodes in ([T] * B, [T, T, 0, max(1, T - 1), T]):
            out, lse, _ = run_tree(c, q, kd, vd, up=dc.words(up), nodes=nodes, cap=cap, workspace=ws)
            check_tree(c, q, kd, vd, out, lse, up=up, nodes=nodes, cap=cap)
            for b in range(B):
                n = torch.isnan(out[b]).any(-1)
                assert torch.equal(n, torch.isnan(lse[b])) and n[nodes[b]:].sum() == 0
            assert torch.isnan(out[0, 0, 1]).all() and torch.isnan(out[1, T - 1]).all() and torch.isnan(out[4, T // 2]).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("T,hq", [(1, 1), (1, 8), (2, 8), (3, 6), (9, 8), (32, 8)])
@pytest.mark.parametrize("cap", [0.0, 6.0])
def test_tree_weighted_mean_of_equal_values(dim, T, hq, cap):
    """Where every key holds the same 8-bit row, the output is that row whatever the probabilities. Tolerance: a
    probability as two bf16 parts is off by 2^-16, its product with the value's scale (or the value as two parts) by another
    2^-16, the sums of up to 200 terms by 200 * 2^-24; the rest of 2^-14 is room."""
    lens = [1, 2, 17, 200]
    c = dc.Cache(lens, 1, dim, store="q8_0", seed=3)
    row = rand(71, 1, 1, dim)
    k = rand(72, 200, 1, dim)
    for b, n in enumerate(lens):
        c.pool.append(0, dc.ints([c.seqs[b]]), dc.ints([0]), dc.ints([n]), dc.ints([0]), n, k[:n].contiguous(), row.expand(n, 1, dim).contiguous())
    q, kd, vd = rand(73, 4, T, hq, dim), rand(74, 4, T, 1, dim), rand(75, 4, T, 1, dim)
    up = [[0] * T for _ in range(4)]
    out, lse, _ = run_tree(c, q, kd, vd, up=dc.words(up), cap=cap, dtype=torch.float32)
    want = c.rows(0)[1][0, 0].double()
    assert ((out.double() - want).abs() <= 2 ** -14 * want.abs()).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("T,hq", [(1, 4), (2, 8), (9, 4), (32, 4)])
def test_tree_values_beyond_their_scale(dim, T, hq):
    """8-bit values whose f16 scale overflowed are infinite (and NaN where the 8 bits are 0): so are the outputs."""
    c = dc.Cache([40, 300], 1, dim, store="q8_0", seed=4)
    big = torch.ones(1, 1, dim, dtype=torch.bfloat16, device="cuda")
    big[0, 0, 5], big[0, 0, 32:64] = 1e8, -1e8
    c.pool.append(0, c.seq_ids, dc.ints([7, 290]), dc.ints([1, 1]), dc.ints([0, 0]), 1, torch.ones_like(big), big)
    q, kd, vd = rand(81, 2, T, hq, dim), rand(82, 2, T, 1, dim), rand(83, 2, T, 1, dim)
    out, lse, _ = run_tree(c, q, kd, vd)
    assert torch.isinf(out[..., 32:64]).all() and torch.isnan(out[..., 6]).all()
    check_tree(c, q, kd, vd, out, lse)


@pytest.mark.parametrize("store,dim", STORES)
@pytest.mark.parametrize("T,hq", [(1, 4), (3, 5), (9, 8)])
def test_key_weights_of_rows_that_do_not_count(store, dim, T, hq):
    """Keys that are not finite get nothing from rows that add nothing: tokens at or above n_nodes, rows with lse -inf, and
    what fills up the kernel's tiles of rows."""
    n = 90
    c = dc.Cache([n, n, n], 1, dim, store=store, seed=2)
    bad = torch.full((3, 1, dim), float("nan"), dtype=torch.bfloat16, device="cuda")
    bad[1], bad[2] = float("inf"), 1e8
    c.pool.append(0, c.seq_ids, dc.ints([4] * 3), dc.ints([3] * 3), dc.ints([0] * 3), 3, bad, bad)
    q = rand(91, 3, T, hq, dim)
    nodes = [0, T, max(0, T - 1)]
    prm = c.pool.tree_params(layer=0, seq_ids=c.seq_ids, n_draft=T, q_heads=hq, scale=0.125, n_nodes=dc.ints(nodes))
    lse = torch.full((3, T, hq), -math.inf, device="cuda")
    lse[:, nodes[2]:] = 1.0  # (only of request 2 are these tokens beyond the last)
    lse[1] = -math.inf
    w = torch.rand(3, 1, n, generator=torch.Generator().manual_seed(1)).cuda()
    old = w.clone()
    c.pool.key_weights(prm, q, lse, w, 1.0)
    torch.cuda.synchronize()
    assert c.pool.status() == 0
    assert torch.equal(w, old)


@pytest.mark.parametrize("dim", [48, 64, 128, 256])
@pytest.mark.parametrize("T,hq", [(1, 3), (5, 3), (17, 2)])
def test_key_weights_of_a_key_far_below(dim, T, hq):
    """A key of -infinity that every row takes to a score of -inf: weight 0, not the 0 * inf of rows that are not there."""
    c = dc.Cache([70], 1, dim, seed=6)
    bad = torch.zeros(1, 1, dim, dtype=torch.bfloat16, device="cuda")
    bad[0, 0, 2] = float("-inf")
    c.pool.append(0, c.seq_ids, dc.ints([9]), dc.ints([1]), dc.ints([0]), 1, bad, bad)
    q = rand(92, 1, T, hq, dim)
    q[..., 2] = 1.0
    prm = c.pool.tree_params(layer=0, seq_ids=c.seq_ids, n_draft=T, q_heads=hq, scale=0.125, n_nodes=dc.ints([T]))
    s = torch.einsum("thd,kd->thk", q[0].double(), c.rows(0)[0][:, 0].double()) * 0.125
    lse = torch.logsumexp(s, -1).float()[None]
    w = torch.zeros(1, 1, 70, device="cuda")
    c.pool.key_weights(prm, q, lse, w, 0.0)
    torch.cuda.synchronize()
    want = torch.exp(s - lse[0].double()[..., None]).sum((0, 1))
    assert want[9] == 0 and w[0, 0, 9] == 0
    assert ((w[0, 0].double() - want).abs() <= 1e-4 * want).all()


@pytest.mark.parametrize("store", ["bf16", "q8_0"])
def test_evict_resize_and_attend_with_a_short_request(store):
    """The whole turn over a batch in which one request has fewer tokens than are kept: it stays as it is, the others are cut,
    and attention sees the rows that stayed and no slot besides. The pages that a request would gain hold NaN."""
    lens, keep = [300, 41, 100, 101], 100
    c = dc.Cache(lens, 2, 64, store=store, block=16, seed=8, spare=8, width=25)
    junk = c.pool.seq_create()
    c.pool.seq_resize(junk, 8 * 16)
    c.pool.sync()
    nan = torch.full((128, 2, 64), float("inf" if store == "q8_0" else "nan"), dtype=torch.bfloat16, device="cuda")
    c.pool.append(0, dc.ints([junk]), dc.ints([0]), dc.ints([128]), dc.ints([0]), 128, nan, nan)
    c.pool.seq_free(junk)
    before = [c.rows(b) for b in range(4)]
    w = torch.rand(1, 4, 2, 300, generator=torch.Generator().manual_seed(5)).cuda()
    kept = torch.empty(1, 4, 2, keep, dtype=torch.int32, device="cuda")
    c.pool.evict_by_weight(0, 1, c.seq_ids, w, keep=keep, first=4, recent=8, kept=kept)
    for b, s in enumerate(c.seqs):
        if c.lens[b] > keep:
            c.pool.seq_resize(s, keep)
            c.lens[b] = keep
    c.pool.sync()
    assert [c.pool.seq_get(s).n_tokens for s in c.seqs] == [100, 41, 100, 100]
    q, kd, vd = rand(101, 4, 3, 4, 64), rand(102, 4, 3, 2, 64), rand(103, 4, 3, 2, 64)
    out, lse, _ = run_tree(c, q, kd, vd)
    check_tree(c, q, kd, vd, out, lse)
    for b in range(4):  # and the rows in use are those that were kept
        for x, y in zip(before[b], c.rows(b)):
            for h in range(2):
                at = kept[0, b, h, :c.lens[b]].long()
                assert torch.equal(y[:, h], x[at, h])


def test_evict_beside_a_sequence_beyond_the_limit():
    """A sequence longer than any eviction takes, which the call does not name, changes nothing; named, it is reported."""
    n = ekv.MAX_EVICT_TOKENS + 1
    c = dc.Cache([300, n, 90], 1, 16, block=256, seed=3)
    w = torch.rand(1, 2, 1, 300, generator=torch.Generator().manual_seed(6)).cuda()
    kept = torch.empty(1, 2, 1, 80, dtype=torch.int32, device="cuda")
    c.pool.evict_by_weight(0, 1, dc.ints([c.seqs[0], c.seqs[2]]), w, keep=80, first=4, recent=8, kept=kept)
    torch.cuda.synchronize()
    assert c.pool.status() == 0
    for b, m in enumerate((300, 90)):
        assert kept[0, b, 0].tolist() == dc.evict(w[0, b, 0, :m].tolist(), m, 80, 4, 8)
    long = torch.rand(1, 1, 1, n, generator=torch.Generator().manual_seed(7)).cuda()
    c.pool.evict_by_weight(0, 1, dc.ints([c.seqs[1]]), long, keep=80, first=4, recent=8, kept=kept)
    torch.cuda.synchronize()
    assert c.pool.status() == ekv.DEV_ERR_BAD_POS


@pytest.mark.parametrize("lens", [[1100, 4096], [4097, 300], [16384, 16385, 16383, 200]])
@pytest.mark.parametrize("stride", [0, 21000])
def test_evict_rows_shorter_than_what_is_read_ahead(lens, stride):
    """Rows on both sides of what the selection holds in registers, with strides as long as the rows and longer, beside an idle
    sequence that is longer still."""
    c = dc.Cache(lens, 1, 16, block=256, seed=4, spare=84, width=84)
    c.pool.seq_resize(c.pool.seq_create(), 20500)
    c.pool.sync()
    w = torch.rand(1, len(lens), 1, max(max(lens), stride), generator=torch.Generator().manual_seed(9)).cuda()
    w[..., ::5] = 0.5
    pos = torch.arange(w.shape[-1], dtype=torch.int32, device="cuda").flip(0).repeat(1, len(lens), 1, 1).contiguous()
    check_evict(c, w, 150, 4, 20)
    check_evict(c, w, 1000, 4, 20, positions=pos, seen=[w.shape[-1]] * len(lens))


def test_rope_is_ready_when_it_is_made():
    """A handle's frequencies are on the device when the call that makes it returns, whatever stream uses them first."""
    c = dc.Cache([64], 1, 256, seed=1)
    q, pos, out = rand(111, 32, 4, 256), dc.ints(range(32)), torch.empty(32, 4, 256, dtype=torch.bfloat16, device="cuda")
    n, at = dc.ints([32]), dc.ints([0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for i in range(50):
        rope = ekv.Rope(rotary_dims=256, freq_base=100.0 + i)
        c.pool.rope_append(rope, 0, None, None, n, at, 32, pos, q=q, q_out=out, stream=side)
        side.synchronize()
        want, size = dc.rope(q, pos, dc.rope_table(256, 100.0 + i), 256, False)
        close_turned(out, want, size)
        rope.close()


def test_tree_calls_that_start_under_one_another():
    """Calls of many rows over pools of several widths, a hundred in a row without a wait between them (each kernel starts while
    the one before it drains, and holds tensor memory of its own): every result is that of the call alone."""
    calls = []
    for store, dim, T in (("bf16", 64, 6), ("bf16", 256, 6), ("q8_0", 128, 6), ("bf16", 64, 40), ("bf16", 128, 6), ("q8_0", 64, 40)):
        c = dc.Cache([200, 90, 0], 2, dim, store=store, seed=dim)
        q, kd, vd = rand(121, 3, T, 8, dim), rand(122, 3, T, 2, dim), rand(123, 3, T, 2, dim)
        for ws in (False, True):
            out, lse, prm = run_tree(c, q, kd, vd, workspace=ws)
            room = torch.empty(c.pool.tree_attention_workspace_size(prm), dtype=torch.uint8, device="cuda") if ws else None
            calls.append((c, prm, q, kd, vd, torch.zeros_like(out), torch.zeros_like(lse), room, out, lse))
    for _ in range(10):
        for c, prm, q, kd, vd, out, lse, room, _, _ in calls:
            c.pool.tree_attention(prm, q, kd, vd, out, lse, room)
    torch.cuda.synchronize()
    for c, prm, q, kd, vd, out, lse, room, want, want_lse in calls:
        assert c.pool.status() == 0 and torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("heads", [2 ** 13, 2 ** 29, 2 ** 30, 2 ** 31 - 1])
def test_rope_refuses_heads_beyond_its_divisions(heads):
    """Nothing is launched for head counts whose items are beyond the kernel's 32-bit divisions, also where the check's own
    product would pass 64 bits."""
    c = dc.Cache([4], 1, 16, seed=1)
    rope, one, q = ekv.Rope(rotary_dims=16), dc.ints([0]), torch.zeros(64, dtype=torch.bfloat16, device="cuda")
    code = ekv.lib.ekv_rope_append(c.pool.h, rope.h, 0, 1, None, None, one.data_ptr(), one.data_ptr(), 1, one.data_ptr(), heads,
                                   q.data_ptr(), 0, q.data_ptr(), None, None, 0, None)
    assert code == ekv.ERR_UNSUPPORTED


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("T,hq", [(1, 4), (20, 4), (40, 4)])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_tree_capped_scores_of_infinity(dim, T, hq, sign):
    """cap * tanh takes an infinite product to -cap or cap, a score like any other: where every visible key has it the output
    is the values' mean and lse is that score plus the logarithm of their number."""
    lens = [70, 1, 640, 5000]
    c = dc.Cache(lens, 1, dim, seed=7)
    q, kd, vd = rand(171, 4, T, hq, dim), rand(172, 4, T, 1, dim), rand(173, 4, T, 1, dim)
    q[..., 3] = sign
    k = rand(174, max(lens), 1, dim)
    k[..., 3] = kd[..., 3] = float("inf")
    v = rand(175, max(lens), 1, dim)
    for b, n in enumerate(lens):
        c.pool.append(0, dc.ints([c.seqs[b]]), dc.ints([0]), dc.ints([n]), dc.ints([0]), n, k, v)
    up = [[1 << t if t % 2 else 0 for t in range(T)] for _ in range(4)]
    for ws in (True, False):
        out, lse, _ = run_tree(c, q, kd, vd, up=dc.words(up), cap=5.0, workspace=ws)
        check_tree(c, q, kd, vd, out, lse, up=up, cap=5.0)
        for b, n in enumerate(lens):
            for t in range(T):
                want = sign * 5.0 + math.log(n + t % 2)
                assert ((lse[b, t] - want).abs() < 1e-4).all()


@pytest.mark.parametrize("store,dim", STORES)
@pytest.mark.parametrize("T,hq", [(1, 1), (1, 8), (3, 4), (5, 4), (9, 4), (40, 4)])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_tree_f32_outputs(store, dim, T, hq, cap):
    """An f32 output is more than a bf16 one with zeros behind it. Tolerance, of A = sum p |v|: a probability as two bf16 parts
    is off by 2^-16, over 8-bit pages its product with the value's scale, or the value as two parts, by another 2^-16 (2^-14
    leaves twice that), sums of n terms by n 2^-24, and an error e of a score moves numerator and denominator by e: head_dim *
    2^-24 * sum |q k|, and 2e-5 for cap and exponential."""
    lens = [1, 2, 5, 300, 2500]
    c = dc.Cache(lens, 1, dim, store=store, block=32, seed=dim)
    q, kd, vd = rand(191, 5, T, hq, dim), rand(192, 5, T, 1, dim), rand(193, 5, T, 1, dim)
    up = [dc.tree_words(T, b) for b in range(5)]
    for ws in (True, False):
        out, _, _ = run_tree(c, q, kd, vd, up=dc.words(up), cap=cap, dtype=torch.float32, workspace=ws)
        for b, n in enumerate(lens):
            k, v = c.rows(b)
            want, _, size, most = dc.tree_attention(q[b], k, v, kd[b], vd[b], up[b], T, 1 / math.sqrt(dim), cap)
            e = dim * 2 ** -24 * most + 2e-5
            off = (out[b].double() - want).abs() - size * (2 ** -14 + (n + T) * 2 ** -24 + 2 * e[..., None])
            assert not (off > 0).any(), (b, ((out[b].double() - want).abs() / size).max().item())


@pytest.mark.parametrize("store", ["bf16", "q8_0"])
@pytest.mark.parametrize("rotary", [64, 34, 18])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_has_one_rounding(store, rotary, interleaved):
    """A turned value has the same bits whichever form of the kernel turns it: out of place, in place, and on the way into the
    pages (40 million values: of those whose last bit of f32 hangs on the order of the products, some fall on a bf16 tie)."""
    n, heads, dim = 4000, 4, 64
    pools = []
    for _ in range(2):
        p = ekv.Pool(dtype=ekv.DTYPE_Q8_0 if store == "q8_0" else ekv.DTYPE_BF16, block_tokens=16, n_blocks=250, kv_heads=heads, head_dim=dim,
                     max_seqs=1, max_blocks_per_seq=250)
        p.seq_resize(p.seq_create(), n)
        p.sync()
        pools.append(p)
    rope, zero, count = ekv.Rope(rotary_dims=rotary, interleaved=interleaved), dc.ints([0]), dc.ints([n])
    size = n * heads * (dim * 2 if store == "bf16" else dim // 32 * 34)
    g = torch.Generator("cuda").manual_seed(rotary)
    for _ in range(40):
        k = torch.randn(n, heads, dim, device="cuda", generator=g).bfloat16()
        pos = torch.randint(0, 1 << 20, (n,), device="cuda", dtype=torch.int32, generator=g)
        out, there = torch.empty_like(k), k.clone()
        pools[0].rope_append(rope, 0, zero, zero, count, zero, n, pos, q=k, q_out=out, k=k, v=k)
        pools[0].rope_append(rope, 0, None, None, count, zero, n, pos, q=there, q_out=there)
        pools[1].append(0, zero, zero, count, zero, n, out, k)
        assert torch.equal(out.view(torch.int16), there.view(torch.int16))
        got, want = ([torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2)] for _ in range(2))
        pools[0].gather(0, 0, 0, n, ekv.GATHER_NATIVE, *got)
        pools[1].gather(0, 0, 0, n, ekv.GATHER_NATIVE, *want)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_evict_leaves_what_it_reports():
    """A sequence that the call cannot cut keeps its weights and positions also where the outputs are the inputs; the others of
    the call are cut."""
    c = dc.Cache([100, 70, 90], 1, 64, seed=1)
    w = torch.rand(1, 3, 1, 95, generator=torch.Generator().manual_seed(2)).cuda()  # (the first is longer than that)
    pos = torch.arange(95, dtype=torch.int32, device="cuda").repeat(1, 3, 1, 1).contiguous()
    old, rows = w.clone(), [c.rows(b) for b in range(3)]
    kept = torch.zeros(1, 3, 1, 60, dtype=torch.int32, device="cuda")
    ids = dc.ints([c.seqs[0], c.seqs[1], 999])
    c.pool.evict_by_weight(0, 1, ids, w, keep=60, first=2, recent=5, kept=kept, weights_out=w, positions=pos, positions_out=pos)
    torch.cuda.synchronize()
    assert c.pool.status() in (ekv.DEV_ERR_BAD_POS, ekv.DEV_ERR_BAD_SEQ)
    for b in (0, 2):
        assert (kept[0, b] == -1).all() and torch.equal(w[0, b], old[0, b]) and pos[0, b, 0].tolist() == list(range(95))
        for x, y in zip(rows[b], c.rows(b)):
            assert torch.equal(x, y)
    want = dc.evict(old[0, 1, 0, :70].tolist(), 70, 60, 2, 5)
    assert kept[0, 1, 0].tolist() == want and torch.equal(w[0, 1, 0, :60], old[0, 1, 0][torch.tensor(want, device="cuda")])
