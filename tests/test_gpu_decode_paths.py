"""Decoding operators on paths that small calls do not take: more requests than a block has threads, workspaces that do not
suffice, two streams at once, graphs replayed at other lengths, and the streaming example along branches that it accepts.
Checks and tolerances are those of test_gpu_decode.py."""
import math

import numpy as np
import pytest
import torch

import decode_cases as dc
import ekv
from test_gpu_decode import check_tree, rand, run_tree
from test_gpu_streaming_example import example, prompts, turn

pytestmark = pytest.mark.gpu


def ragged(n, seed, most=200):
    """Lengths of n requests; the ones around the sizes of a block (160 to 384 threads) are empty or short, as are the last."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, most, n)
    lens[rng.random(n) < 0.2] = 0
    for at in (160, 192, 256, 320, 352, 384, 480):
        lens[max(0, at - 2):at + 2] = [0, 1, 0, 65][:len(lens[max(0, at - 2):at + 2])]
    lens[-1] = 0
    lens[n // 3] = 3000  # (long enough for the call to be cut into parts)
    return [int(x) for x in lens]


@pytest.mark.parametrize("n", [161, 320, 500])
@pytest.mark.parametrize("store,dim,T,hq", [("bf16", 64, 1, 4), ("q8_0", 128, 2, 4), ("bf16", 64, 6, 4), ("bf16", 128, 5, 32), ("q8_0", 64, 9, 4)])
def test_more_requests_than_threads(n, store, dim, T, hq):
    """Few rows (one per KV head and more), many rows on either tile form, with 8-bit pages too; the key weights of the same
    call."""
    lens = ragged(n, n + T)
    c = dc.Cache(lens, 1, dim, store=store, block=16, seed=n)
    q, kd, vd = rand(131, n, T, hq, dim), rand(132, n, T, 1, dim), rand(133, n, T, 1, dim)
    nodes = [T if b % 3 else max(0, T - b % 5) for b in range(n)]
    out, lse, prm = run_tree(c, q, kd, vd, nodes=nodes)
    check_tree(c, q, kd, vd, out, lse, nodes=nodes)
    w = torch.full((n, 1, 3008), 0.25, device="cuda")
    c.pool.key_weights(prm, q, lse, w, 1.0)
    torch.cuda.synchronize()
    assert c.pool.status() == 0
    for b in range(n):
        m = lens[b]
        assert (w[b, 0, m:] == 0.25).all()
        if m and nodes[b]:
            s, size = dc.tree_scores(q[b, :nodes[b]].double(), c.rows(b)[0].double(), 1 / math.sqrt(dim), 0.0)
            got = torch.exp(s - lse[b, :nodes[b]].double()[..., None]).sum((0, 1))
            tol = got * (dim * 2 ** -24 * size.max().item() + 2e-5) + (got + 0.25) * 1e-6
            assert ((w[b, 0, :m].double() - 0.25 - got).abs() <= tol).all()
        elif m:
            assert (w[b, 0, :m] == 0.25).all()


@pytest.mark.parametrize("store,dim,T,hq", [("bf16", 128, 1, 8), ("bf16", 64, 20, 4), ("q8_0", 256, 3, 8), ("q8_0", 128, 20, 4)])
def test_tree_workspaces_of_every_size(store, dim, T, hq):
    """A workspace one byte too small, of a few bytes or of none counts as none; nothing outside a given one is written."""
    c = dc.Cache([3000, 40, 0, 700], 1, dim, store=store, seed=2)
    q, kd, vd = rand(141, 4, T, hq, dim), rand(142, 4, T, 1, dim), rand(143, 4, T, 1, dim)
    _, _, prm = run_tree(c, q, kd, vd, workspace=False)
    size = c.pool.tree_attention_workspace_size(prm)
    for given in (0, 16, size - 1, size, size + 160):
        buf = torch.full((size + 1024,), 205, dtype=torch.uint8, device="cuda")
        out, lse = torch.full_like(q, 9.0), torch.full((4, T, hq), 9.0, device="cuda")
        c.pool.tree_attention(prm, q, kd, vd, out, lse, buf[256:256 + given])
        torch.cuda.synchronize()
        assert c.pool.status() == 0
        assert (buf[:256] == 205).all() and (buf[256 + given:] == 205).all()
        if given < size:
            assert (buf == 205).all()
        check_tree(c, q, kd, vd, out, lse)


@pytest.mark.parametrize("store,dim,T,hq", [("bf16", 128, 1, 8), ("bf16", 64, 20, 4), ("q8_0", 256, 3, 8), ("q8_0", 128, 20, 4)])
@pytest.mark.parametrize("workspace", [True, False])
def test_tree_prefixes_beyond_or_below_what_was_said(store, dim, T, hq, workspace):
    """max_prefix picks how the work is shared and nothing else: far too small, right and far too large, beside an idle
    sequence that is longer than all."""
    c = dc.Cache([2100, 40, 0, 700], 1, dim, store=store, block=64, seed=2, spare=160, width=160)
    c.pool.seq_resize(c.pool.seq_create(), 10000)
    c.pool.sync()
    q, kd, vd = rand(181, 4, T, hq, dim), rand(182, 4, T, 1, dim), rand(183, 4, T, 1, dim)
    for said in (0, 1, 100, 700, 2100, 2 ** 31 - 1):
        prm = c.pool.tree_params(layer=0, seq_ids=c.seq_ids, n_draft=T, q_heads=hq, scale=1 / math.sqrt(dim), max_prefix=said)
        room = torch.empty(c.pool.tree_attention_workspace_size(prm), dtype=torch.uint8, device="cuda") if workspace else None
        out, lse = torch.full_like(q, 9.0), torch.full((4, T, hq), 9.0, device="cuda")
        c.pool.tree_attention(prm, q, kd, vd, out, lse, room)
        w = torch.zeros(4, 1, 2100, device="cuda")
        c.pool.key_weights(prm, q, lse, w, 0.0)
        torch.cuda.synchronize()
        assert c.pool.status() == 0
        check_tree(c, q, kd, vd, out, lse)
        for b, n in enumerate(c.lens):
            s, _ = dc.tree_scores(q[b].double(), c.rows(b)[0].double(), 1 / math.sqrt(dim), 0.0)
            want = torch.exp(s - lse[b].double()[..., None]).sum((0, 1))
            assert ((w[b, 0, :n].double() - want).abs() <= 1e-4 * want).all() and (w[b, 0, n:] == 0).all()


def test_two_streams_with_workspaces_of_their_own():
    """Calls of two pools, and of one pool, side by side on two streams: the bits of the calls alone."""
    calls = []
    for store, dim, T in (("bf16", 128, 1), ("bf16", 64, 20), ("q8_0", 128, 2), ("q8_0", 64, 40)):
        c = dc.Cache([4000, 900, 0], 2, dim, store=store, seed=dim + T)
        q, kd, vd = rand(151, 3, T, 8, dim), rand(152, 3, T, 2, dim), rand(153, 3, T, 2, dim)
        out, lse, prm = run_tree(c, q, kd, vd)
        w = torch.zeros(3, 2, 4000, device="cuda")
        c.pool.key_weights(prm, q, lse, w, 0.0)
        calls.append((c, prm, q, kd, vd, out, lse, w))
    streams = [torch.cuda.Stream() for _ in range(2)]
    mine = []
    for s in streams:
        for c, prm, q, kd, vd, out, lse, w in calls:
            room = torch.empty(c.pool.tree_attention_workspace_size(prm), dtype=torch.uint8, device="cuda")
            mine.append((s, torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(w), room))
    torch.cuda.synchronize()
    for _ in range(5):
        for i, (c, prm, q, kd, vd, *_) in enumerate(calls):
            for j in range(2):
                s, out, lse, w, room = mine[j * len(calls) + i]
                c.pool.tree_attention(prm, q, kd, vd, out, lse, room, stream=s)
                c.pool.key_weights(prm, q, lse, w, 0.0, stream=s)
    torch.cuda.synchronize()
    for i, (c, _, _, _, _, out, lse, w) in enumerate(calls):
        assert c.pool.status() == 0
        for j in range(2):
            _, o, l, x, _ = mine[j * len(calls) + i]
            assert torch.equal(o, out) and torch.equal(l, lse) and torch.equal(x, w)


@pytest.mark.parametrize("store,dim,T,hq", [("bf16", 64, 1, 4), ("bf16", 128, 9, 4), ("q8_0", 128, 1, 4), ("q8_0", 64, 9, 4)])
@pytest.mark.parametrize("first", [[100, 700], [5000, 20000]])
def test_graphs_at_other_lengths(store, dim, T, hq, first):
    """Attention, key weights and eviction captured at some lengths and replayed at others, shorter and far longer, empty ones
    and ones past what the eviction read ahead at its capture among them."""
    most = 21000
    c = dc.Cache([most, most], 1, dim, store=store, block=64, seed=5)
    q, kd, vd = rand(161, 2, T, hq, dim), rand(162, 2, T, 1, dim), rand(163, 2, T, 1, dim)
    keep = 64
    gen = torch.Generator().manual_seed(3)
    old = torch.rand(1, 2, 1, most, generator=gen).cuda()
    w, out, lse = old.clone(), torch.zeros_like(q), torch.zeros(2, T, hq, device="cuda")
    kept = torch.zeros(1, 2, 1, keep, dtype=torch.int32, device="cuda")
    prm = c.pool.tree_params(layer=0, seq_ids=c.seq_ids, n_draft=T, q_heads=hq, scale=1 / math.sqrt(dim))
    ws = torch.empty(c.pool.tree_attention_workspace_size(prm), dtype=torch.uint8, device="cuda")

    def resize(lens):
        for s, n in zip(c.seqs, lens):
            c.pool.seq_resize(s, n)
        c.pool.sync()
        c.lens = list(lens)

    def calls():
        c.pool.tree_attention(prm, q, kd, vd, out, lse, ws)
        c.pool.key_weights(prm, q, lse, w[0], 0.5)
        c.pool.evict_by_weight(0, 1, c.seq_ids, w, keep=keep, first=4, recent=8, kept=kept)

    tables = [c.pool.seq_get(s).blocks for s in c.seqs]
    resize(first)
    calls()  # (kernels are loaded before the capture)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        calls()
    for lens in (first, [0, 65], [20999, 3], [640, 16385], [64, 20]):
        resize([0, 0])
        for s, t, n in zip(c.seqs, tables, lens):
            c.pool.seq_set_blocks(s, t, n)
        resize(lens)
        w.copy_(old)
        before = [c.rows(b) for b in range(2)]
        g.replay()
        torch.cuda.synchronize()
        assert c.pool.status() == 0
        for b, n in enumerate(lens):
            k, v = before[b]
            up = [(2 << t) - 1 for t in range(T)]
            want, want_lse, size, _ = dc.tree_attention(q[b], k, v, kd[b], vd[b], up, T, 1 / math.sqrt(dim), 0.0)
            assert ((out[b].double() - want).abs() <= 1.25 * 2 ** -7 * size + 1e-30).all()
            assert ((lse[b].double() - want_lse).abs() <= 1e-4 * (1 + want_lse.abs())).all()
            s, _ = dc.tree_scores(q[b].double(), k.double(), 1 / math.sqrt(dim), 0.0) if n else (None, None)
            if n:
                x = torch.exp(s - lse[b].double()[..., None]).sum((0, 1)) + 0.5 * old[0, b, 0, :n].double()
                assert ((w[0, b, 0, :n].double() - x).abs() <= 1e-4 * x).all()
            assert torch.equal(w[0, b, 0, n:], old[0, b, 0, n:])
            assert kept[0, b, 0].tolist() == dc.evict(w[0, b, 0, :n].tolist(), n, keep, 4, 8)
            m = min(n, keep)
            at = kept[0, b, 0, :m].long()
            for x, y in zip(before[b], c.rows(b)):
                assert torch.equal(y[:m], x[at])


@pytest.mark.parametrize("q8", [False, True])
def test_example_takes_branches_of_unequal_lengths(q8):
    """Stream.step with trees of which each request accepts another path, one along a second branch and one of the root alone:
    the cached rows are those of the accepted tokens at their positions, and the next step's logits are those of the text."""
    ex = example()
    model = ex.Decoder()
    stream = ex.Stream(3, 400, 256, store=ekv.DTYPE_Q8_0 if q8 else ekv.DTYPE_BF16)
    texts = prompts(ex, 3, 21)
    stream.step(model, [t[:20] for t in texts])
    #        0 root; 1, 2, 3 a chain under it; 4, 5 a second branch under the root; 6 under 1
    words = [1, 0b11, 0b111, 0b1111, 0b10001, 0b110001, 0b1000011]
    paths = [[0, 4, 5], [0], [0, 1, 6]]
    tokens = [[t[20]] + [(7 * i + 31 * j) % ex.VOCAB for j in range(1, 7)] for i, t in enumerate(texts)]
    stream.step(model, tokens, [words] * 3, lambda logits: paths)
    for i, p in enumerate(paths):
        texts[i] = texts[i][:20] + [tokens[i][j] for j in p]
    assert stream.cached == stream.seen == [23, 21, 23] and stream.pool.status() == 0
    for i, text in enumerate(texts):
        n = len(text)
        pos = torch.arange(n, device="cuda")
        for h in range(ex.KV_HEADS):
            assert stream.positions[0, i, h, :n].tolist() == list(range(n))
        k, v = (torch.empty(n, ex.KV_HEADS, ex.DIM, device="cuda") for _ in range(2))
        stream.pool.gather(0, stream.seqs[i], 0, n, ekv.GATHER_F32, k, v)
        rows = (ex.norm(model.embed[torch.tensor(text, device="cuda")]) @ model.qkv[0]).view(n, -1, ex.DIM)
        want_k, want_v = turn(rows[:, ex.Q_HEADS:ex.Q_HEADS + ex.KV_HEADS], pos), rows[:, -ex.KV_HEADS:].double()
        for got, want in ((k, want_k), (v, want_v)):
            top = want.abs().view(n, ex.KV_HEADS, -1, 32).amax(-1, keepdim=True).expand(-1, -1, -1, 32).reshape(want.shape)
            size = (want ** 2 + want.roll(ex.DIM // 2, -1) ** 2).sqrt()
            assert ((got.double() - want).abs() <= size * 2 ** -7 + 1e-3 + (top / 250 if q8 else 0)).all()


def test_example_accepts_guesses_that_come_true():
    """Guesses that are the decoder's own next tokens are taken: far fewer steps than tokens, and the same text."""
    ex = example()
    model = ex.Decoder()
    plain, _ = ex.generate(model, ex.Stream(2, 400, 256), prompts(ex, 2, 30), 48, 1)
    stream = ex.Stream(2, 400, 256)
    real = ex.guesses
    try:
        def told(text, n):
            whole = next(p for p in plain if p[:30] == text[:30])
            ahead = whole[len(text):len(text) + n - 1]
            if len(text) > len(whole) - n or whole[:len(text)] != text:
                return real(text, n)
            return [text[-1]] + ahead, [(2 << j) - 1 for j in range(len(ahead) + 1)]

        ex.guesses = told
        texts, steps = ex.generate(model, stream, prompts(ex, 2, 30), 48, 6)
    finally:
        ex.guesses = real
    assert stream.pool.status() == 0 and steps < 40
    for text, p in zip(texts, plain):
        assert len(text) >= 78
