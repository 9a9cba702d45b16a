"""Windowed attention on the GPU: how calls are shared over the SMs. The formula and its tolerances are those of test_gpu_window.py."""
import math
import os
import subprocess
import sys

import pytest
import torch

import decode_cases as dc
import ekv
from test_gpu_window import Call, formula, rand, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store,dim", [("bf16", 64), ("bf16", 128), ("q8_0", 128), ("q8_0", 256)])
def test_ranges_of_whole_units(store, dim):
    """Far more units than CTAs, of lengths that differ, with empty requests, one row, and rows that end inside a row tile."""
    rows = [(31 * i) % 70 for i in range(170)]
    past = [(197 * i) % 900 for i in range(170)]
    call = Call(past, rows, 8, 4, dim, store=store, window=200, sinks=4, seed=dim)
    assert sum(1 for r in rows if r) * 4 > 4 * 148
    out = call.run()
    call.check(out, requests=range(0, 170, 3))
    assert torch.equal(call.run(workspace=False), out)


@pytest.mark.parametrize("store,dim", [("bf16", 128), ("bf16", 256), ("q8_0", 64)])
def test_ranges_with_several_row_tiles(store, dim):
    rows = [300 - 7 * i for i in range(40)]
    call = Call([11 * i for i in range(40)], rows, 16, 4, dim, store=store, window=77, seed=dim + 1)
    call.check(call.run(), requests=range(0, 40, 5))


def test_cut_units_of_many_ctas():
    """One long unit's tiles over every CTA, several row tiles and heads, and rows of the last tile alone."""
    for store, dim, rows, hq, hk in (("bf16", 128, 33, 8, 1), ("bf16", 64, 257, 3, 3), ("q8_0", 128, 100, 8, 2), ("q8_0", 256, 18, 1, 1)):
        call = Call([9000, 0, 4000], [rows, 1, rows], hq, hk, dim, store=store, seed=rows, block=64)
        call.check(call.run())


def test_more_requests_than_ranges_look_through():
    past = [(7 * i) % 30 for i in range(4200)]
    call = Call(past, [3] * 4200, 8, 1, 64, window=20, sinks=2, seed=3)
    out = call.run()
    call.check(out, requests=[0, 1, 31, 32, 2099, 4094, 4095, 4096, 4097, 4199])
    assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("store,dim", [("bf16", 128), ("bf16", 256), ("q8_0", 256)])
@pytest.mark.parametrize("n", [1, 13, 17, 37, 75, 150])
def test_clusters_in_one_turn_and_more(store, dim, n):
    """Single tokens of as many requests as leave each cluster size its place, and a ragged end."""
    past = [1000 + (89 * i) % 300 for i in range(n)]
    call = Call(past, [1] * n, 8, 1, dim, store=store, window=1000, sinks=4, seed=n)
    for ws in (True, False):
        call.check(call.run(ws), requests=sorted({0, 1, n // 2, n - 1} & set(range(n))))


@pytest.mark.parametrize("rows", [1, 12, 200])
def test_two_calls_at_once(rows):
    """Two streams, a workspace each."""
    calls = [Call([1500, 3, 700], [rows] * 3, 8, 2, 128, window=w, sinks=4, seed=w) for w in (0, 333)]
    want = [c.run() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    prms, outs, ws = [], [], []
    for c in calls:
        prms.append(c.c.pool.window_params(layer=0, seq_ids=c.c.seq_ids, dst_pos=dc.ints(c.past), n_rows=c.n_rows, src_row=c.src, max_rows=rows,
                                           q_heads=8, scale=1 / math.sqrt(128), window=c.window, sinks=4))
        outs.append(torch.zeros_like(c.q))
        ws.append(torch.empty(c.c.pool.window_attention_workspace_size(prms[-1]), dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, prm, out, w, s in zip(calls, prms, outs, ws, streams):
            c.c.pool.window_attention(prm, c.q, out, w, stream=s)
    torch.cuda.synchronize()
    for out, x, c in zip(outs, want, calls):
        assert torch.equal(out, x) and c.c.pool.status() == 0


@pytest.mark.parametrize("store,rows", [("bf16", 1), ("q8_0", 1), ("bf16", 40)])
def test_replayed_as_the_cache_grows(store, rows):
    """A graph captured over a short cache, replayed when the sequences are far longer."""
    lens = [200, 2500, 3]
    call = Call([n - rows if n > rows else 0 for n in lens], [min(rows, n) for n in lens], 8, 1, 128, store=store, window=1200, sinks=4, seed=4,
                width=400, spare=10)
    pool, full = call.c.pool, call.c.rows(1)
    for s, n in zip(call.c.seqs, lens):
        pool.seq_resize(s, min(n, 50))
    pool.sync()
    dst = dc.ints([max(0, min(n, 50) - rows) for n in lens])
    prm = pool.window_params(layer=0, seq_ids=call.c.seq_ids, dst_pos=dst, n_rows=call.n_rows, src_row=call.src, max_rows=rows, q_heads=8,
                             scale=1 / math.sqrt(128), window=1200, sinks=4)
    ws = torch.empty(pool.window_attention_workspace_size(prm), dtype=torch.uint8, device="cuda")
    out, stream = torch.zeros_like(call.q), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        pool.window_attention(prm, call.q, out, ws)
    graph.replay()
    torch.cuda.synchronize()
    k, v = (x[:min(lens[1], 50)] for x in full)
    n = int(call.n_rows[1])
    s = int(call.src[1])
    want, size, most = formula(call.q[s:s + n], k, v, 50 - n, 1200, 4)
    assert ((out[s:s + n].double() - want).abs() <= tolerance(store, call.many, size, most)).all()
    # back to the full length: the rows are appended again
    for q, n in zip(call.c.seqs, lens):
        pool.seq_resize(q, n)
    pool.sync()
    kk, vv = (x.bfloat16() for x in full)
    pool.append(0, call.c.seq_ids[1:2], dc.ints([0]), dc.ints([2500]), dc.ints([0]), 2500, kk, vv)
    dst.copy_(dc.ints([n - r for n, r in zip(lens, [min(rows, n) for n in lens])]))
    graph.replay()
    torch.cuda.synchronize()
    n = int(call.n_rows[1])
    k, v = call.c.rows(1)
    want, size, most = formula(call.q[s:s + n], k, v, 2500 - n, 1200, 4)
    assert ((out[s:s + n].double() - want).abs() <= tolerance(store, call.many, size, most)).all()
    assert pool.status() == 0


def test_same_sequence_twice_and_out_of_order():
    """Two requests of one sequence (chunks that follow one another), their rows in another order in q."""
    call = Call([60, 0, 300], [60, 60, 60], 4, 2, 64, window=90, sinks=3, seed=8)
    call.check(call.run())
    seqs = dc.ints([call.c.seqs[2], call.c.seqs[2], call.c.seqs[0]])
    dst, src = dc.ints([300, 240, 60]), dc.ints([120, 0, 60])
    out = call.run(seq_ids=seqs, dst_pos=dst, src_row=src)
    k, v = call.c.rows(2)
    for at, past, kk, vv in ((120, 300, k, v), (0, 240, k[:300], v[:300])):
        want, size, most = formula(call.q[at:at + 60], kk, vv, past, 90, 3)
        assert ((out[at:at + 60].double() - want).abs() <= tolerance("bf16", True, size, most)).all()
    assert call.c.pool.status() == 0


def test_scores_far_apart():
    """Scores that climb by hundreds along the cache, and rows that see only the smallest of them: the reference maximum moves in
    every tile, and later in none."""
    for rows in (1, 40):
        for turn in (1.0, -1.0):
            call = Call([700], [rows], 4, 1, 128, window=0, seed=2, scale=0.1)
            k = torch.zeros(700 + rows, 1, 128)
            k[:, 0, 0] = torch.linspace(0, 40, 700 + rows) * turn
            v = rand(5, 700 + rows, 1, 128)
            call.q.zero_()
            call.q[:, :, 0] = 150.0
            call.c.pool.append(0, call.c.seq_ids, dc.ints([0]), dc.ints([700 + rows]), dc.ints([0]), 700 + rows, k.bfloat16().cuda(), v)
            kk, vv = call.c.rows(0)
            out = call.run()
            want, size, most = formula(call.q, kk, vv, 700, 0, 0)
            # f32 sums of products up to M are off by 2^-24 of it for each of log2(128) + 1 steps and the scale: 2^-20 M, twice
            tol = tolerance("bf16", call.many, size, most) + torch.expm1(most * 2 ** -19) * size
            assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("store", ["bf16", "q8_0"])
@pytest.mark.parametrize("rows", [1, 50])
def test_the_largest_windows_and_first_tokens(store, rows):
    """Windows and numbers of first tokens up to what their type holds: every slot up to the row's own."""
    call = Call([300, 0], [rows, rows], 4, 2, 64, store=store, window=0, seed=6)
    want = call.run()
    call.check(want)
    for window, sinks in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (0, 2 ** 31 - 1), (5, 2 ** 31 - 1), (1, 100000)):
        got = call.run(window=window, sinks=sinks)
        call.check(got)


CAPTURE_FIRST = """
import math, sys
import torch
import decode_cases as dc, ekv
from test_gpu_window import Call
rows, dim, store = int(sys.argv[1]), int(sys.argv[2]), sys.argv[3]
call = Call([1500, 900], [rows, rows], 8, 1, dim, store=store, window=1200, sinks=4)
prm = call.c.pool.window_params(layer=0, seq_ids=call.c.seq_ids, dst_pos=dc.ints(call.past), n_rows=call.n_rows, src_row=call.src, max_rows=rows,
                                q_heads=8, scale=1 / math.sqrt(dim), window=1200, sinks=4)
ws = torch.empty(call.c.pool.window_attention_workspace_size(prm), dtype=torch.uint8, device="cuda")
out, s = torch.zeros_like(call.q), torch.cuda.Stream()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    call.c.pool.window_attention(prm, call.q, out, ws)
g.replay()
torch.cuda.synchronize()
call.check(out)
assert torch.equal(out, call.run())
print("done")
"""


@pytest.mark.parametrize("rows,dim,store", [(1, 256, "bf16"), (1, 128, "q8_0"), (60, 128, "bf16")])
def test_the_first_call_of_a_process_is_captured(rows, dim, store):
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(os.path.abspath(ekv.__file__)), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-c", CAPTURE_FIRST, str(rows), str(dim), store], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("store,dim", [("bf16", 128), ("q8_0", 256)])
def test_an_idle_sequence_far_longer(store, dim, rows):
    """The longest live sequence stands for the call's where max_len is not given: work is shared for 6000 slots, then for the call's own."""
    call = Call([700, 30, 300], [rows] * 3, 8, 2, dim, store=store, sinks=4, width=400, spare=400)
    call.check(call.run())
    idle = call.c.pool.seq_create()
    call.c.pool.seq_resize(idle, 6000)
    call.c.pool.sync()
    for max_len in (0, 700 + rows, 31):
        for ws in (True, False):
            call.check(call.run(ws, max_len=max_len))
