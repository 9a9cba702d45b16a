"""Windowed attention on the GPU against the formula in 64 bits.

Tolerances, of A = sum p |v| (p the softmax weights). An output is rounded to bf16: half a step, 2^-8 of it. bf16 pages: each
probability is rounded so too, and so is their sum: a weight is off by at most twice 2^-8. f32 scores and exponentials: 2^-12 covers
head_dim * 2^-24 of sum |q k| here. 8-bit pages, up to 16 rows of a KV head: two bf16 parts, 2^-15. More rows: f16 operands, 2^-11 each
in the value, twice in the weight, and 2^-11 of M = max sum |q k| in a score, which moves a weight by e^(2 * that) at most."""
import math

import pytest
import torch

import decode_cases as dc
import ekv

pytestmark = pytest.mark.gpu


def rand(seed, *shape, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).bfloat16().cuda()


def seen(past, n, window, sinks, first=0, rows=None):
    """Which slots [rows, past + n] the rows from `first` on see."""
    p = past + first + torch.arange(n - first if rows is None else rows, device="cuda")[:, None]
    k = torch.arange(past + n, device="cuda")[None]
    return (k <= p) & ((k > p - window) | (k < sinks)) if window else k <= p


def formula(q, k, v, past, window, sinks):
    """out, A and M of one request: q [rows, heads, dim], k, v [slots, kv_heads, dim]."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out, size, most = (torch.zeros(n, hq, m, dtype=torch.float64, device="cuda") for m in (d, d, 1))
    for r0 in range(0, n, 256):
        rows = min(256, n - r0)
        see = seen(past, n, window, sinks, r0, rows)
        for h in range(hq):
            kk, vv = k[:, h // group], v[:, h // group]
            x = (q[r0:r0 + rows, h] @ kk.T / math.sqrt(d)).masked_fill(~see, -math.inf)
            p = torch.softmax(x, -1)
            out[r0:r0 + rows, h] = p @ vv
            size[r0:r0 + rows, h] = p @ vv.abs()
            a = (q[r0:r0 + rows, h].abs() @ kk.abs().T / math.sqrt(d)).masked_fill(~see, 0)
            most[r0:r0 + rows, h, 0] = a.amax(-1)
    return out, size, most


def tolerance(store, many, size, most):
    if store == "bf16":
        return (3 * 2 ** -8 + 2 ** -12) * size + 1e-30
    if not many:
        return (2 ** -8 + 2 ** -12) * size + 1e-30
    return (2 ** -8 + 5 * 2 ** -11 + torch.expm1(2 * 2 ** -11 * most)) * size + 1e-30


class Call:
    def __init__(self, past, rows, hq, hk, dim, *, store="bf16", block=16, window=0, sinks=0, seed=0, scale=1.5, stride=0, **kw):
        self.past, self.rows, self.store, self.window, self.sinks, self.hq = past, rows, store, window, sinks, hq
        self.c = dc.Cache([p + n for p, n in zip(past, rows)], hk, dim, store=store, block=block, seed=seed, **kw)
        self.total = sum(rows)
        wide = rand(seed + 1, max(1, self.total), hq * dim + stride, scale=scale)
        self.q = wide[:, :hq * dim].unflatten(1, (hq, dim))
        n = dc.ints(rows)
        self.n_rows, self.src = n, (n.cumsum(0) - n).int()
        self.many = max(rows) * (hq // hk) > 16

    def run(self, workspace=True, stream=None, max_len=0, **kw):
        arg = dict(layer=0, seq_ids=self.c.seq_ids, dst_pos=dc.ints(self.past), n_rows=self.n_rows, src_row=self.src, max_rows=max(self.rows),
                   q_heads=self.hq, scale=1 / math.sqrt(self.q.shape[2]), window=self.window, sinks=self.sinks, max_len=max_len)
        arg.update(kw)
        prm = self.c.pool.window_params(**arg)
        behind = torch.full((self.q.shape[0] + 3, *self.q.shape[1:]), 7.0, dtype=torch.bfloat16, device="cuda")
        out = behind[:self.q.shape[0]]
        ws = torch.full((self.c.pool.window_attention_workspace_size(prm),), 255, dtype=torch.uint8, device="cuda") if workspace else None
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        self.c.pool.window_attention(prm, self.q, out, ws, stream=stream)
        torch.cuda.synchronize()
        assert (behind[self.q.shape[0]:] == 7.0).all()
        return out

    def check(self, out, requests=None):
        for b, (past, n) in enumerate(zip(self.past, self.rows)):
            if n == 0 or (requests is not None and b not in requests):
                continue
            k, v = self.c.rows(b)
            s = int(self.src[b])
            want, size, most = formula(self.q[s:s + n], k, v, past, self.window, self.sinks)
            got = out[s:s + n].double()
            bad = (got - want).abs() > tolerance(self.store, self.many, size, most)
            assert torch.isfinite(got).all() and not bad.any(), (b, (got - want).abs().max().item(), bad.nonzero()[:3].tolist(), int(bad.sum()))
        assert self.c.pool.status() == 0


STORES = [("bf16", 64), ("bf16", 128), ("bf16", 256), ("q8_0", 64), ("q8_0", 128), ("q8_0", 256)]


@pytest.mark.parametrize("store,dim", STORES)
@pytest.mark.parametrize("hq,hk", [(4, 4), (8, 1), (6, 2)])
def test_single_tokens(store, dim, hq, hk):
    """Caches from nothing to several tiles; windows from one slot to none; first tokens inside and before the window."""
    past = [0, 1, 63, 64, 333, 1000]
    for window, sinks in ((0, 0), (1, 0), (64, 4), (100, 13), (300, 350), (7, 1)):
        call = Call(past, [1] * 6, hq, hk, dim, store=store, window=window, sinks=sinks, seed=dim + window)
        for ws in (True, False):
            call.check(call.run(ws))


@pytest.mark.parametrize("store,dim", STORES)
@pytest.mark.parametrize("rows,hq,hk", [(2, 8, 2), (5, 6, 2), (16, 1, 1), (17, 2, 2), (33, 8, 1), (70, 4, 1), (129, 3, 3), (300, 2, 1)])
def test_chunks(store, dim, rows, hq, hk):
    """Ragged chunks after caches of any length, empty ones and requests without rows among them."""
    past, n = [0, 517, 40, 0, 5], [rows, rows - 1, max(1, rows // 2), 0, 1]
    for window, sinks in ((0, 0), (24, 5), (200, 66)):
        call = Call(past, n, hq, hk, dim, store=store, window=window, sinks=sinks, seed=rows + dim, block=24)
        for ws in (True, False):
            call.check(call.run(ws))


@pytest.mark.parametrize("block", [8, 16, 24, 40, 128, 256])
@pytest.mark.parametrize("store", ["bf16", "q8_0"])
def test_blocks(store, block):
    for rows in (1, 37):
        call = Call([515, 200, 63], [rows] * 3, 8, 2, 128, store=store, block=block, window=100, sinks=20, seed=block)
        call.check(call.run())


@pytest.mark.parametrize("store,dim,hq,hk", [("bf16", 64, 4, 2), ("bf16", 128, 8, 2), ("bf16", 256, 4, 1), ("q8_0", 128, 4, 1), ("q8_0", 256, 8, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (256, 4), (1000, 130)])
def test_prompts(store, dim, hq, hk, window, sinks):
    """Whole prompts of many tiles with scores that rise and fall, and a chunk at the end of a long cache."""
    call = Call([0, 0, 2900], [1500, 777, 130], hq, hk, dim, store=store, window=window, sinks=sinks, seed=3, scale=4.0, block=64)
    for ws in (True, False):
        call.check(call.run(ws))


def test_many_units_go_round():
    """More units than CTAs, of very different lengths, in whole units and cut ones."""
    rows = [7 + 61 * i % 500 for i in range(40)]
    call = Call([3 * i for i in range(40)], rows, 8, 4, 64, window=0, seed=5)
    call.check(call.run())
    call = Call([900 * (i % 2) for i in range(90)], [1] * 90, 8, 4, 128, store="q8_0", window=333, sinks=4, seed=6)
    call.check(call.run())


@pytest.mark.parametrize("rows", [1, 2, 60])
def test_strided_queries_and_given_length(rows):
    """q as a slice of a projection; max_len below and above the call's lengths; an idle sequence far longer."""
    call = Call([700, 30], [rows, rows], 8, 2, 128, window=200, sinks=4, stride=256, width=400)
    out = call.run()
    call.check(out)
    for max_len in (1, 100, 1 << 30):
        call.check(call.run(max_len=max_len))
    idle = call.c.pool.seq_create()
    call.c.pool.seq_resize(idle, 32)
    call.c.pool.sync()
    call.check(call.run())


@pytest.mark.parametrize("store,dim", [("bf16", 64), ("bf16", 128), ("bf16", 256)])
@pytest.mark.parametrize("rows,hq", [(1, 8), (7, 2), (40, 4), (300, 1)])
def test_hidden_values_do_not_leak(store, dim, rows, hq):
    """Infinite and NaN keys and values outside a row's view do not reach it, and inside it do: behind the window, between the first
    tokens and the window, after the row, past the sequence's end."""
    past, n, window, sinks = 330, rows, 90, 3
    call = Call([past], [n], hq, 1, dim, store=store, window=window, sinks=sinks, seed=9)
    end = past + n
    k, v = (x.bfloat16() for x in call.c.rows(0))
    marks = {2: math.inf, 3: math.nan, 5: -math.inf, 200: math.nan, past - window: math.inf, past - 20: math.inf, end - 1: math.nan}
    if n > 5:
        marks.update({past + 2: -math.inf, past + 4: math.nan, end - 2: math.inf})
    cols = {}
    for i, (slot, x) in enumerate(sorted(marks.items())):
        cols[slot] = (7 * i) % dim
        v[slot, 0, cols[slot]] = x
        if slot in (3, 200):
            k[slot] = x  # a key that nobody in the call sees
    call.c.pool.append(0, call.c.seq_ids, dc.ints([0]), dc.ints([end]), dc.ints([0]), end, k, v)
    for ws in (True, False):
        out = call.run(ws)
        fixed = v.clone()
        fixed[~torch.isfinite(fixed)] = 0
        safe = k.clone()
        safe[~torch.isfinite(safe)] = 0
        want, size, most = formula(call.q, safe, fixed, past, window, sinks)
        see = seen(past, n, window, sinks)
        extra = torch.zeros(n, dim, dtype=torch.float64, device="cuda")
        for slot, x in marks.items():
            extra[see[:, slot], cols[slot]] += x
        want = want + extra[:, None]
        got = out.double()
        fine = torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
        assert ((got - want).abs() <= tolerance(store, call.many, size, most))[fine].all()
        assert call.c.pool.status() == 0


@pytest.mark.parametrize("store", ["bf16", "q8_0"])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_bad_requests_are_zero_and_reported(store, rows):
    past, n = [100, 200, 300, 64], [rows] * 4
    call = Call(past, n, 4, 2, 64, store=store, window=50, sinks=2)
    ids = [call.c.seqs[0], 77, call.c.seqs[2], call.c.seqs[3]]
    for ws in (True, False):
        out = call.run(ws, seq_ids=dc.ints(ids))
        assert call.c.pool.status() == ekv.DEV_ERR_BAD_SEQ
        s = [int(x) for x in call.src]
        assert (out[s[1]:s[1] + rows] == 0).all()
        call.check(out, requests=[0, 2, 3])
        out = call.run(ws, dst_pos=dc.ints([100, 200, 301, -1]))
        assert call.c.pool.status() == ekv.DEV_ERR_BAD_POS
        assert (out[s[2]:] == 0).all()
        call.check(out, requests=[0, 1])


def test_rows_beyond_max_rows_stay():
    call = Call([50, 10], [9, 9], 4, 1, 64)
    out = torch.full_like(call.q, 5.0)
    prm = call.c.pool.window_params(layer=0, seq_ids=call.c.seq_ids, dst_pos=dc.ints([50, 10]), n_rows=call.n_rows, src_row=call.src, max_rows=4,
                                    q_heads=4, scale=0.125)
    call.c.pool.window_attention(prm, call.q, out)
    assert (out[4:9] == 5.0).all() and (out[13:] == 5.0).all() and not (out[:4] == 5.0).all()


@pytest.mark.parametrize("store,dim,rows", [("bf16", 128, 1), ("bf16", 128, 300), ("q8_0", 256, 40), ("q8_0", 64, 1)])
def test_streams_graphs_and_repeated_calls(store, dim, rows):
    """The same bits on another stream, replayed, and with a dirty workspace; two graphs with one workspace, one after the other."""
    call = Call([2000, 77], [rows, rows], 8, 1, dim, store=store, window=1500, sinks=4)
    want = call.run()
    assert torch.equal(call.run(), want)
    assert torch.equal(call.run(stream=torch.cuda.Stream()), want)
    prm = call.c.pool.window_params(layer=0, seq_ids=call.c.seq_ids, dst_pos=dc.ints(call.past), n_rows=call.n_rows, src_row=call.src, max_rows=rows,
                                    q_heads=8, scale=1 / math.sqrt(dim), window=1500, sinks=4)
    ws = torch.full((call.c.pool.window_attention_workspace_size(prm),), 255, dtype=torch.uint8, device="cuda")
    outs, graphs, s = [torch.zeros_like(call.q) for _ in range(2)], [], torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call.c.pool.window_attention(prm, call.q, o, ws)
            call.c.pool.window_attention(prm, call.q, o, ws)
        graphs.append(g)
    for g in graphs * 2:
        g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    assert call.c.pool.status() == 0


def test_values_beyond_f16():
    """8-bit pages with many rows compute in f16: a query, or a block, beyond its range is reported."""
    call = Call([40], [30], 4, 1, 64, store="q8_0")
    call.q[3, 1, 5] = 1e5
    call.run()
    assert call.c.pool.status() == ekv.DEV_ERR_F16_RANGE
    call = Call([40], [30], 4, 1, 64, store="q8_0")
    k, v = rand(1, 1, 1, 64), rand(2, 1, 1, 64)
    v[0, 0, 9] = 1e6
    call.c.pool.append(0, call.c.seq_ids, dc.ints([7]), dc.ints([1]), dc.ints([0]), 1, k, v)
    call.run()
    assert call.c.pool.status() == ekv.DEV_ERR_F16_RANGE


@pytest.mark.parametrize("dim,rows,hq", [(64, 20, 1), (128, 3, 8), (256, 40, 1)])
@pytest.mark.parametrize("below", [14.0, 18.0, 19.5])
def test_many_small_keys_behind_a_heavy_one(dim, rows, hq, below):
    """8-bit pages, many rows: the output is made of probabilities far below the row's largest, whose value is 0. P is f16 with 7 bits of
    headroom: a key is off by half of the smallest step at most, 2^-25 of 2^7, 2^-32 of the row's largest, beside the relative terms
    (values are at most 1)."""
    past = 60000
    call = Call([past], [rows], hq, 1, dim, store="q8_0", block=64, seed=1)
    n = past + rows
    k, v = torch.zeros(n, 1, dim, device="cuda").bfloat16(), torch.ones(n, 1, dim, device="cuda").bfloat16()
    k[0, 0, 3] = 1.0
    v[0] = 0.0
    v[n // 2:] = -0.5
    call.c.pool.append(0, call.c.seq_ids, dc.ints([0]), dc.ints([n]), dc.ints([0]), n, k, v)
    call.q.zero_()
    call.q[:, :, 3] = below * math.sqrt(dim)
    kk, vv = call.c.rows(0)
    want, size, most = formula(call.q, kk, vv, past, 0, 0)
    for ws in (True, False):
        got = call.run(ws).double()
        assert call.c.pool.status() == 0
        tol = (2 ** -8 + 5 * 2 ** -11) * size + torch.expm1(2 * 2 ** -11 * most) * size + n * 2 ** -32
        err = (got - want).abs()
        assert (err <= tol).all()


class Bytes:
    def __init__(self, pool):
        self.__cuda_array_interface__ = dict(shape=(int(pool.info().bytes_prefix),), typestr="|u1", version=2, data=(int(pool.info().prefix_base), False))


def set_scale(call, kv, slot, group, value):
    """The stored scale of 32 values of K (0) or V (1): a pool of one layer and KV head."""
    pool, dim, bt = call.c.pool, call.c.dim, call.c.block
    block = pool.seq_get(call.c.seqs[0]).blocks[slot // bt]
    at = (2 * block + kv) * (bt * dim // 32 * 34) + bt * dim + (slot % bt * (dim // 32) + group) * 2
    torch.as_tensor(Bytes(pool), device="cuda")[at:at + 2] = torch.tensor([value], dtype=torch.float16, device="cuda").view(torch.uint8)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,hq", [(1, 8), (7, 2), (40, 4), (300, 1)])
@pytest.mark.parametrize("window,sinks", [(90, 3), (93, 0), (320, 5), (331, 8), (1, 0)])
def test_hidden_scales_do_not_leak(dim, rows, hq, window, sinks):
    """Infinite and NaN scales of 8-bit rows that no query row sees reach neither the output nor the status: between the first tokens and
    the window, next to them and far from them."""
    past = 335
    call = Call([past], [rows], hq, 1, dim, store="q8_0", window=window, sinks=sinks, seed=9)
    hidden = [s for s in range(past + rows) if sinks <= s <= past - window]
    want = [call.run(ws) for ws in (True, False)]
    assert call.c.pool.status() == 0
    for i, slot in enumerate(sorted(set(hidden[:9] + hidden[::17] + hidden[-9:]))):
        for kv in range(2):
            set_scale(call, kv, slot, (i + kv) % (dim // 32), (math.inf, math.nan, -math.inf, 6e4, math.nan)[(i + kv) % 5])
    rows_now = [x[hidden] for x in call.c.rows(0)]
    assert not hidden or not any(torch.isfinite(x).all() for x in rows_now)
    for ws, x in zip((True, False), want):
        assert torch.equal(call.run(ws), x)
        assert call.c.pool.status() == 0


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,hq", [(1, 8), (7, 2), (4, 4), (40, 4), (300, 1)])
@pytest.mark.parametrize("scale", [math.inf, -math.inf, math.nan])
def test_values_with_scales_that_are_not_finite(dim, rows, hq, scale):
    """They reach the rows that see them and no others. With many rows they count as 0 and are reported."""
    past, window, sinks = 330, 90, 3
    call = Call([past], [rows], hq, 1, dim, store="q8_0", window=window, sinks=sinks, seed=10)
    end = past + rows
    want = [call.run(ws) for ws in (True, False)]
    see = seen(past, rows, window, sinks)
    last = dim // 32 - 1
    slots = {2: 0, past - 20: 1, past - window + 3: 0, past - window + 1: last, end - 1: 1}
    if rows > 3:
        slots[past + 3] = last
    hit = torch.zeros(rows, dim, dtype=torch.bool, device="cuda")
    keys, fixed = call.c.rows(0)
    exact_v = fixed.clone()
    for slot, group in slots.items():
        set_scale(call, 1, slot, group, scale)
        columns = slice(32 * group, 32 * group + 32)
        hit[see[:, slot], columns] = True
        exact_v[slot, 0, columns] = 0
    assert hit.any() and not hit.all() or dim == 64
    exact, size, most = formula(call.q, keys, exact_v, past, window, sinks)
    for ws, x in zip((True, False), want):
        got = call.run(ws)
        status = call.c.pool.status()
        if call.many:
            assert status == ekv.DEV_ERR_F16_RANGE
            bad = (got.double() - exact).abs() > tolerance("q8_0", True, size, most)
            assert torch.isfinite(got).all() and not bad.any()
        else:
            assert status == 0
            assert torch.isfinite(got).logical_not().eq(hit[:, None]).all()
        assert torch.equal(got.masked_fill(hit[:, None], 0), x.masked_fill(hit[:, None], 0))
