"""The pages' operators as a language backbone runs them, one after the other: normed and rotated rows into the pages, windowed
attention, forks that share blocks and go on by themselves, blocks behind the window dropped, rows compacted. Each sequence's rows are
kept beside the pool as plain tensors, and every step's attention is the formula over those (test_gpu_window.py has the tolerances)."""
import math

import pytest
import torch

import decode_cases as dc
import ekv
from test_gpu_window import formula, rand, tolerance

pytestmark = pytest.mark.gpu

LAYERS, HQ, HK, BLOCK, WINDOW, SINKS = 2, 8, 2, 16, 60, 16


class Backbone:
    def __init__(self, store, dim):
        self.store, self.dim = store, dim
        dtype = ekv.DTYPE_BF16 if store == "bf16" else ekv.DTYPE_Q8_0
        self.pool = ekv.Pool(device=0, dtype=dtype, block_tokens=BLOCK, n_blocks=120, kv_heads=HK, head_dim=dim, n_layers=LAYERS, max_seqs=12,
                             max_blocks_per_seq=30)
        self.rope = ekv.Rope(rotary_dims=dim)
        self.norm = [ekv.HeadNorm(q_weight=rand(layer, dim), k_weight=rand(9 + layer, dim)) for layer in range(LAYERS)]
        self.kept = {}  # sequence -> per layer [k, v], the rows that its pages stand for
        self.tokens = {}  # sequence -> tokens so far, dropped ones too
        self.seed = 0

    def add(self):
        s = self.pool.seq_create()
        empty = torch.zeros(0, HK, self.dim, device="cuda")
        self.kept[s], self.tokens[s] = [[empty, empty] for _ in range(LAYERS)], 0
        return s

    def rows_of(self, s, layer):
        n = self.pool.seq_get(s).n_tokens
        out = [torch.zeros(n, HK, self.dim, device="cuda") for _ in range(2)]
        self.pool.gather(layer, s, 0, n, ekv.GATHER_F32, *out)
        return out

    def step(self, seqs, n):
        """n tokens of each sequence."""
        pool, dim, total = self.pool, self.dim, n * len(seqs)
        at = [pool.seq_get(s).n_tokens for s in seqs]
        for s, a in zip(seqs, at):
            pool.seq_resize(s, a + n)
        pool.sync()
        ids, dst, n_rows, src = dc.ints(seqs), dc.ints(at), dc.ints([n] * len(seqs)), dc.ints([n * i for i in range(len(seqs))])
        positions = dc.ints([self.tokens[s] + i for s in seqs for i in range(n)])
        for layer in range(LAYERS):
            self.seed += 1
            q, k, v = rand(self.seed, total, (HQ + 2 * HK) * dim).unflatten(1, (-1, dim)).split([HQ, HK, HK], 1)
            turned, out = torch.empty(total, HQ, dim, dtype=torch.bfloat16, device="cuda"), torch.zeros(total, HQ, dim, dtype=torch.bfloat16, device="cuda")
            pool.norm_rope_append(self.rope, self.norm[layer], layer, ids, dst, n_rows, src, n, positions, q=q, q_out=turned, k=k, v=v)
            prm = pool.window_params(layer=layer, seq_ids=ids, dst_pos=dst, n_rows=n_rows, src_row=src, max_rows=n, q_heads=HQ,
                                     scale=1 / math.sqrt(dim), window=WINDOW, sinks=SINKS)
            ws = torch.empty(pool.window_attention_workspace_size(prm), dtype=torch.uint8, device="cuda")
            pool.window_attention(prm, turned, out, ws)
            for i, (s, a) in enumerate(zip(seqs, at)):
                kk, vv = self.rows_of(s, layer)
                old = self.kept[s][layer]
                assert torch.equal(kk[:a], old[0]) and torch.equal(vv[:a], old[1]), (layer, s)  # no other row has changed
                self.kept[s][layer] = [kk, vv]
                if self.store == "bf16":
                    assert torch.equal(vv[a:].bfloat16(), v[n * i:n * (i + 1)])
                want, size, most = formula(turned[n * i:n * (i + 1)], kk, vv, a, WINDOW, SINKS)
                got = out[n * i:n * (i + 1)].double()
                assert ((got - want).abs() <= tolerance(self.store, n * HQ // HK > 16, size, most)).all(), (layer, s)
        for s in seqs:
            self.tokens[s] += n
        assert pool.status() == 0

    def fork(self, s, n_tokens, count):
        kids = self.pool.seq_fork([s] * count, [n_tokens] * count)
        for kid in kids:
            self.kept[kid] = [[x[:n_tokens].clone() for x in kv] for kv in self.kept[s]]
            self.tokens[kid] = self.tokens[s]
        return kids

    def drop(self, s):
        """Blocks between the first tokens and the window, whole ones."""
        n = self.pool.seq_get(s).n_tokens
        blocks = (n - WINDOW) // BLOCK - 1
        if blocks > 0:
            self.pool.seq_drop_blocks(s, 1, blocks)
            self.kept[s] = [[torch.cat([x[:BLOCK], x[BLOCK * (1 + blocks):]]) for x in kv] for kv in self.kept[s]]
        return max(0, blocks)

    def compact(self, s, slots):
        n = self.pool.seq_get(s).n_tokens
        self.pool.seq_own(s, 0, n)
        self.pool.compact(0, LAYERS, dc.ints([s]), dc.ints([slots]), dc.ints([len(slots)]))
        self.pool.seq_resize(s, len(slots))
        self.pool.sync()
        self.kept[s] = [[x[slots] for x in kv] for kv in self.kept[s]]

    def check(self):
        for s, layers in self.kept.items():
            for layer, kv in enumerate(layers):
                for x, y in zip(self.rows_of(s, layer), kv):
                    assert torch.equal(x, y), (s, layer)
        assert self.pool.status() == 0


@pytest.mark.parametrize("store,dim", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("q8_0", 64), ("q8_0", 128), ("q8_0", 256)])
def test_prompts_forks_and_long_answers(store, dim):
    b = Backbone(store, dim)
    first, second = b.add(), b.add()
    b.step([first], 75)           # a prompt of some blocks and a part of one
    b.step([second], 16)          # exactly one block
    kids = b.fork(first, 75, 3) + b.fork(second, 16, 1) + b.fork(first, 30, 1)
    b.check()
    everyone = [first, second] + kids
    b.step(everyone, 1)
    b.step(everyone[::-1], 5)     # chunks, their rows in another order
    b.pool.seq_free(first)        # its blocks live on in its forks
    del b.kept[first]
    everyone.remove(first)
    dropped = 0
    for i in range(60):
        b.step(everyone, 1)
        if i % 9 == 8:
            dropped += sum(b.drop(s) for s in everyone)
    assert dropped > 6
    b.check()
    grand = b.fork(kids[0], b.pool.seq_get(kids[0]).n_tokens - 7, 2)
    n = b.pool.seq_get(grand[0]).n_tokens
    b.compact(grand[0], list(range(0, 20)) + list(range(21, n, 2)))
    b.step([grand[1], grand[0]], 2)
    b.step(grand + everyone[:2], 1)
    b.check()
    for s in list(b.kept):
        b.pool.seq_free(s)
    assert b.pool.info().free_blocks == 120
