"""Forked sequences and compacted rows on the GPU: bytes against the bytes they came from."""
import numpy as np
import pytest
import torch

import decode_cases as dc
import ekv

pytestmark = pytest.mark.gpu


def rand(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


def cache(lens, hk, dim, *, spare=20, sequences=8, **kw):
    """dc.Cache with room for more sequences and blocks."""
    c = dc.Cache(lens, hk, dim, spare=spare, **kw)
    if sequences:
        # (the pool of dc.Cache has one sequence more than it fills: forks need others)
        p = c.pool
        big = ekv.Pool(device=0, dtype=p.cfg.dtype, block_tokens=p.cfg.block_tokens, n_blocks=p.cfg.n_blocks, kv_heads=hk, head_dim=dim,
                       n_layers=p.cfg.n_layers, max_seqs=len(lens) + sequences, max_blocks_per_seq=p.cfg.max_blocks_per_seq + 2)
        for s in c.seqs:
            v = p.seq_get(s)
            big.seq_set_blocks(big.seq_create(), v.blocks, v.n_tokens)
        big.sync()
        arena(big).copy_(arena(p))
        c.pool = big
    return c


class Memory:
    def __init__(self, pointer, shape, kind):
        self.__cuda_array_interface__ = dict(shape=shape, typestr=kind, version=2, data=(int(pointer), False))


def arena(pool):
    return torch.as_tensor(Memory(pool.info().prefix_base, (pool.info().bytes_prefix,), "|u1"), device="cuda")


def bytes_of(pool, layer, seq, n):
    c = pool.cfg
    size = n * c.kv_heads * (c.head_dim * 2 if c.dtype == ekv.DTYPE_BF16 else c.head_dim // 32 * 34)
    out = [torch.zeros(size + 16, dtype=torch.uint8, device="cuda") for _ in range(2)]
    if n:
        pool.gather(layer, seq, 0, n, ekv.GATHER_NATIVE, *out)
    torch.cuda.synchronize()
    return torch.cat([x[:size] for x in out])


STORES = [("bf16", 48, 16), ("bf16", 64, 24), ("bf16", 256, 64), ("q8_0", 32, 8), ("q8_0", 96, 16), ("q8_0", 128, 40), ("q8_0", 256, 256)]


@pytest.mark.parametrize("store,dim,block", STORES)
def test_forks_hold_what_their_parents_hold(store, dim, block):
    lens = [5 * block + 3, 2 * block, block - 1, 1]
    c = cache(lens, 2, dim, store=store, block=block, layers=3, sequences=12)
    p, before = c.pool, arena(c.pool).clone()
    parents = [0, 0, 1, 2, 3, 0, 0]
    tokens = [lens[0], lens[0], lens[1], lens[2], 1, 2 * block + block // 2, 0]
    kids = p.seq_fork(parents, tokens)
    want = {(layer, s): bytes_of(p, layer, s, lens[s]) for layer in range(3) for s in range(4)}
    for kid, parent, n in zip(kids, parents, tokens):
        v, u = p.seq_get(kid), p.seq_get(parent)
        assert v.n_tokens == n and v.blocks[:n // block] == u.blocks[:n // block]
        for layer in range(3):
            got = bytes_of(p, layer, kid, n)
            row = len(want[layer, parent]) // 2 // lens[parent]
            kv = want[layer, parent].view(2, -1)[:, :n * row].reshape(-1)
            assert torch.equal(got, kv), (kid, layer)
    # nothing else of the pool has changed: only rows of the children's own blocks
    own = {p.seq_get(k).blocks[-1] for k, n in zip(kids, tokens) if n % block}
    per = p.cfg.n_blocks
    tile = arena(p).numel() // 1
    size = int(p.info().block_bytes)
    for layer in range(3):
        for b in range(per):
            at = (layer * per + b) * size
            if b not in own:
                assert torch.equal(arena(p)[at:at + size], before[at:at + size])
    assert tile >= 3 * per * size and p.status() == 0


def test_many_forks_in_one_call():
    """More children than one launch takes, of several parents."""
    c = cache([33, 40, 17], 1, 64, block=16, layers=2, spare=700, sequences=700)
    p = c.pool
    parents = [i // 201 for i in range(603)]
    tokens = [33 - i % 3 if i < 201 else 40 if i < 402 else 17 for i in range(603)]
    kids = p.seq_fork(parents, tokens)
    assert len(set(kids)) == 603
    for i in (0, 1, 200, 201, 255, 256, 401, 402, 511, 512, 602):
        for layer in range(2):
            n = tokens[i]
            a, b = bytes_of(p, layer, kids[i], n).view(2, -1), bytes_of(p, layer, parents[i], c.lens[parents[i]]).view(2, -1)
            assert torch.equal(a, b[:, :a.shape[1]])
    for k in kids:
        p.seq_free(k)
    assert p.info().free_blocks == p.cfg.n_blocks - sum(-(-n // 16) for n in c.lens)


@pytest.mark.parametrize("store", ["bf16", "q8_0"])
def test_writes_to_shared_blocks_are_refused(store):
    """Appends go on in blocks of their own; rows of a shared block are reported and stay, until the sequence owns it."""
    c = cache([40], 1, 64, store=store, block=16, layers=1)
    p = c.pool
    kid, = p.seq_fork([0], [40])
    rope = ekv.Rope(rotary_dims=64)
    norm = ekv.HeadNorm()
    k, v = rand(1, 20, 1, 64), rand(2, 20, 1, 64)

    def put(how, seq, pos, n):
        ids, one = dc.ints([seq]), dc.ints([0])
        if how == "append":
            p.append(0, ids, dc.ints([pos]), dc.ints([n]), one, n, k, v)
        elif how == "rope":
            p.rope_append(rope, 0, ids, dc.ints([pos]), dc.ints([n]), one, n, dc.ints(range(20)), k=k, v=v)
        else:
            p.norm_rope_append(rope, norm, 0, ids, dc.ints([pos]), dc.ints([n]), one, n, dc.ints(range(20)), k=k, v=v)
        return p.status()

    for seq in (0, kid):
        before = bytes_of(p, 0, seq, 40).view(2, -1)
        for how in ("append", "rope", "norm"):
            assert put(how, seq, 30, 1) == ekv.DEV_ERR_BAD_BLOCK, how
            assert put(how, seq, 0, 16) == ekv.DEV_ERR_BAD_BLOCK, how
            assert put(how, seq, 32, 8) == 0, how  # the last block is its own
        row = before.shape[1] // 40
        assert torch.equal(bytes_of(p, 0, seq, 40).view(2, -1)[:, :32 * row], before[:, :32 * row])
    # a compaction into a shared block is refused, one inside the sequence's own block is not
    assert (p.compact(0, 1, dc.ints([kid]), dc.ints([[5, 6]]), dc.ints([2])), p.status())[1] == ekv.DEV_ERR_BAD_BLOCK
    keep = dc.ints([list(range(33)) + [36]])
    assert (p.compact(0, 1, dc.ints([kid]), keep, dc.ints([34])), p.status())[1] == 0
    # grown past the shared part, each in new blocks
    for seq in (0, kid):
        p.seq_resize(seq, 60)
    p.sync()
    assert put("append", 0, 40, 20) == 0
    mine = bytes_of(p, 0, 0, 60)
    assert put("rope", kid, 40, 20) == 0
    assert torch.equal(bytes_of(p, 0, 0, 60), mine)
    # one owns the first block, then both may write theirs
    p.seq_own(kid, 3, 4)
    assert put("append", kid, 0, 16) == 0 and torch.equal(bytes_of(p, 0, 0, 60), mine)
    assert put("append", kid, 16, 1) == ekv.DEV_ERR_BAD_BLOCK
    assert put("append", 0, 0, 16) == 0  # (the other's last holder)
    p.seq_free(kid)
    assert put("append", 0, 16, 16) == ekv.DEV_ERR_BAD_BLOCK  # not known to the device before the next sync, or own
    p.seq_own(0, 16, 16)
    assert put("append", 0, 16, 16) == 0


def test_own_copies_many_blocks_of_every_layer():
    c = cache([8 * 300 + 5], 1, 32, store="q8_0", block=8, layers=2, spare=320)
    p = c.pool
    kid, = p.seq_fork([0], [2405])
    want = [bytes_of(p, layer, 0, 2405) for layer in range(2)]
    p.seq_own(kid, 0, 2405)
    a, b = p.seq_get(0).blocks, p.seq_get(kid).blocks
    assert not set(a) & set(b)
    k, v = rand(3, 2405, 1, 32), rand(4, 2405, 1, 32)
    for layer in range(2):
        assert torch.equal(bytes_of(p, layer, kid, 2405), want[layer])
        p.append(layer, dc.ints([0]), dc.ints([0]), dc.ints([2405]), dc.ints([0]), 2405, k, v)
        assert p.status() == 0
        assert torch.equal(bytes_of(p, layer, kid, 2405), want[layer]) and not torch.equal(bytes_of(p, layer, 0, 2405), want[layer])


def test_own_uploads_the_table():
    """What follows ekv_seq_own sees the sequence's length and blocks, whether or not a block was shared."""
    c = cache([40, 20], 1, 64, block=16, layers=1)
    p = c.pool
    kid, = p.seq_fork([0], [40])
    k, v = rand(1, 30, 1, 64), rand(2, 30, 1, 64)
    for seq, pos, n in ((kid, 40, 30), (0, 40, 5), (1, 20, 28)):
        p.seq_resize(seq, pos + n)
        p.seq_own(seq, pos, n)  # blocks of its own
        p.append(0, dc.ints([seq]), dc.ints([pos]), dc.ints([n]), dc.ints([0]), n, k, v)
        assert p.status() == 0, seq
    p.seq_resize(kid, 75)
    p.seq_own(kid, 75, 0)  # no block at all
    p.append(0, dc.ints([kid]), dc.ints([70]), dc.ints([5]), dc.ints([0]), 5, k, v)
    assert p.status() == 0


def test_evict_with_shared_blocks():
    """Rows move where the sequence owns the blocks they go to; a move into a shared block is reported."""
    c = cache([64], 1, 64, block=16, layers=1)
    p = c.pool
    kid, = p.seq_fork([0], [64])
    w = torch.zeros(1, 1, 1, 64, device="cuda")
    w[..., 40:] = 1.0  # the heaviest rows lie above keep: the holes below are in shared blocks
    kept = torch.empty(1, 1, 1, 32, dtype=torch.int32, device="cuda")
    before = bytes_of(p, 0, 0, 64)
    p.evict_by_weight(0, 1, dc.ints([kid]), w, keep=32, first=0, recent=0, kept=kept)
    assert p.status() == ekv.DEV_ERR_BAD_BLOCK
    assert torch.equal(bytes_of(p, 0, 0, 64), before)
    p.evict_by_weight(0, 1, dc.ints([kid]), 1 - w, keep=40, first=0, recent=0, kept=torch.empty(1, 1, 1, 40, dtype=torch.int32, device="cuda"))
    assert p.status() == 0  # nothing moves
    p.seq_own(kid, 0, 32)
    p.evict_by_weight(0, 1, dc.ints([kid]), w, keep=32, first=0, recent=0, kept=kept)
    assert p.status() == 0 and torch.equal(bytes_of(p, 0, 0, 64), before)
    rows = before.view(2, 64, -1)[:, kept.flatten().long()]
    assert torch.equal(bytes_of(p, 0, kid, 32).view(2, 32, -1), rows)


def kept_slots(n, seed, share):
    rng = np.random.default_rng(seed)
    return [int(x) for x in np.nonzero(rng.random(n) < share)[0]]


@pytest.mark.parametrize("store,dim,block", STORES + [("bf16", 16, 8), ("bf16", 80, 16), ("bf16", 128, 64), ("q8_0", 160, 16), ("q8_0", 224, 24)])
def test_compact(store, dim, block):
    """Rows together in order, in some layers; lists of every kind; rows past them as they were."""
    lens = [3000, 517, 64, 1, 0, 700, 255]
    c = dc.Cache(lens, 2, dim, store=store, block=block, layers=3, seed=dim)
    lists = [kept_slots(3000, 1, 0.7), kept_slots(517, 2, 0.1), list(range(64)), [0], [], [699], list(range(1, 255))]
    stride = max(len(x) for x in lists) + 5
    slots = dc.ints([x + [-9] * (stride - len(x)) for x in lists])
    want = {(i, layer): bytes_of(c.pool, layer, c.seqs[i], n).view(2, n, -1) for i, n in enumerate(lens) if n for layer in range(3)}
    c.pool.compact(1, 2, c.seq_ids, slots, dc.ints([len(x) for x in lists]))
    assert c.pool.status() == 0
    for (i, layer), rows in want.items():
        got = bytes_of(c.pool, layer, c.seqs[i], lens[i]).view(2, lens[i], -1)
        if layer == 0:
            assert torch.equal(got, rows)
            continue
        n = len(lists[i])
        assert torch.equal(got[:, :n], rows[:, lists[i]]), (i, layer)
        assert torch.equal(got[:, n:], rows[:, n:]), (i, layer)


@pytest.mark.parametrize("store,dim", [("bf16", 128), ("q8_0", 256)])
@pytest.mark.parametrize("B,layers,hk,n", [(1, 1, 1, 20000), (9, 4, 8, 3001), (2, 18, 1, 1100)])
def test_compact_few_and_many_strips(store, dim, B, layers, hk, n):
    """One strip of many chunks by a cluster, many strips by one CTA each; a few slots leave, most leave."""
    for share in (0.99, 0.3):
        lens = [n - 7 * b for b in range(B)]
        c = dc.Cache(lens, hk, dim, store=store, block=64, layers=layers, seed=1)
        lists = [kept_slots(m, b, share) for b, m in enumerate(lens)]
        stride = max(len(x) for x in lists)
        slots = dc.ints([x + [0] * (stride - len(x)) for x in lists])
        want = [bytes_of(c.pool, layer, c.seqs[b], lens[b]).view(2, lens[b], -1)[:, lists[b]] for b in range(B) for layer in range(layers)]
        c.pool.compact(0, layers, c.seq_ids, slots, dc.ints([len(x) for x in lists]))
        assert c.pool.status() == 0
        for i, rows in enumerate(want):
            b, layer = i // layers, i % layers
            got = bytes_of(c.pool, layer, c.seqs[b], len(lists[b])).view(2, len(lists[b]), -1)
            assert torch.equal(got, rows), (b, layer)


def test_compact_reports_bad_lists():
    """Entries that are not ascending, not above their place, or not of the sequence are reported and not moved; so are whole
    requests; others of the call are done."""
    lens = [100, 100, 100, 100]
    c = dc.Cache(lens, 1, 64, block=16, seed=4)
    before = [bytes_of(c.pool, 0, s, 100).view(2, 100, -1) for s in c.seqs]

    def run(lists, n_keep, seq_ids=None):
        c.pool.compact(0, 1, c.seq_ids if seq_ids is None else seq_ids, dc.ints(lists), dc.ints(n_keep))
        return c.pool.status()

    good = list(range(10, 20))
    assert run([good[:5] + [14] + good[6:], good, good, good], [10, 0, 101, 0]) == ekv.DEV_ERR_BAD_POS
    now = [bytes_of(c.pool, 0, s, 100).view(2, 100, -1) for s in c.seqs]
    want = before[0].clone()
    for i, s in enumerate(good):
        if i != 5:
            want[:, i] = before[0][:, s]
    assert torch.equal(now[0], want)
    for b in (1, 2, 3):
        assert torch.equal(now[b], before[b])
    assert run([[0, 100], [0, 99], [-1, 3], [1, 5]], [2, 2, 2, 2]) == ekv.DEV_ERR_BAD_POS
    now = [bytes_of(c.pool, 0, s, 100).view(2, 100, -1) for s in c.seqs]
    assert torch.equal(now[0], want) and torch.equal(now[1][:, 1], before[1][:, 99])
    assert torch.equal(now[2][:, 1], before[2][:, 3]) and torch.equal(now[2][:, 0], before[2][:, 0])
    assert torch.equal(now[3][:, :2], before[3][:, [1, 5]])
    assert run([[5, 6]] * 4, [2, 2, 2, -1], dc.ints([c.seqs[0], 99, -1, c.seqs[3]])) in (ekv.DEV_ERR_BAD_SEQ, ekv.DEV_ERR_BAD_POS)
    assert torch.equal(bytes_of(c.pool, 0, c.seqs[0], 2).view(2, 2, -1), want[:, [5, 6]])


def in_place_again(n, **at):
    """0 .. n - 1 with some entries replaced."""
    x = list(range(n))
    for i, s in at.items():
        x[int(i[1:])] = s
    return x


@pytest.mark.parametrize("store", ["bf16", "q8_0"])
@pytest.mark.parametrize("slots", [in_place_again(5, _1=7), [0, 0, 2, 3], [0, 1, 1, 3], in_place_again(5, _0=-2), in_place_again(6, _2=700),
                                   in_place_again(256, _100=650), in_place_again(600, _100=650), in_place_again(600, _101=99, _300=640),
                                   in_place_again(690, _255=256, _256=255), in_place_again(513, _511=2 ** 31 - 1)])
def test_compact_reports_bad_entries_before_rows_in_place(store, slots):
    """An entry that is out of order, or a row that moves before it, is seen where later rows are in their places again."""
    n, lens = len(slots), [700, 700]
    c = dc.Cache(lens, 2, 64, store=store, block=16, layers=2, seed=8)
    before = {(layer, s): bytes_of(c.pool, layer, s, 700).view(2, 700, -1) for layer in range(2) for s in c.seqs}
    good = list(range(0, 2 * n, 2))[:350]
    lists = [slots, good + [0] * (n - len(good))]
    c.pool.compact(0, 2, c.seq_ids, dc.ints(lists), dc.ints([n, len(good[:n])]))
    assert c.pool.status() == ekv.DEV_ERR_BAD_POS
    for (layer, s), rows in before.items():
        want = rows.clone()
        if s == c.seqs[0]:
            for i, x in enumerate(slots):
                if x >= i and x < 700 and x > (slots[i - 1] if i else -1):
                    want[:, i] = rows[:, x]
        else:
            want[:, :len(good[:n])] = rows[:, good[:n]]
        assert torch.equal(bytes_of(c.pool, layer, s, 700).view(2, 700, -1), want)


@pytest.mark.parametrize("n", [0, 1, 255, 256, 257, 4096, 4097, 9000])
@pytest.mark.parametrize("first", [0, 1, 255, 256, 4095, 4096, 8191, 8999])
def test_compact_behind_rows_in_place(n, first):
    """Rows before the first that moves stay, however many they are."""
    c = dc.Cache([10000], 1, 32, store="q8_0", block=64, layers=1, seed=8)
    lists = [i if i < first else i + 3 + i % 7 // 6 for i in range(n)]
    lists = sorted(set(lists))
    rows = bytes_of(c.pool, 0, c.seqs[0], 10000).view(2, 10000, -1)
    c.pool.compact(0, 1, c.seq_ids, dc.ints([lists + [0]]), dc.ints([len(lists)]))
    assert c.pool.status() == 0
    want = rows.clone()
    want[:, :len(lists)] = rows[:, lists]
    assert torch.equal(bytes_of(c.pool, 0, c.seqs[0], 10000).view(2, 10000, -1), want)


def test_compact_replayed_and_on_another_stream():
    c = dc.Cache([600, 300], 2, 128, block=32, layers=2, seed=6)
    lists = [kept_slots(600, 1, 0.8)[:300], kept_slots(300, 2, 0.9)[:200]]
    slots, n_keep = dc.ints([lists[0], lists[1] + [0] * (300 - len(lists[1]))]), dc.ints([len(x) for x in lists])
    want = [bytes_of(c.pool, 1, s, n).view(2, n, -1) for s, n in zip(c.seqs, c.lens)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        c.pool.compact(0, 2, c.seq_ids, slots, n_keep)
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        rows = want[i].clone()
        for _ in range(2):
            rows[:, :len(lists[i])] = rows[:, lists[i]].clone()
        assert torch.equal(bytes_of(c.pool, 1, c.seqs[i], c.lens[i]).view(2, c.lens[i], -1), rows)
    assert c.pool.status() == 0
